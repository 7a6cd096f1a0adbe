// Library-wide runtime pieces of the C ABI: version, error strings, launch
// accounting.  The device error word lives with the kernels that set it
// (attention.cu).
#include <atomic>
#include <cstdio>

#include "common.cuh"
#include "tc.cuh"

namespace vdit {

__device__ int g_wait_check_error = 0;

namespace {

constexpr int kErrWaitCheck = 0x5754;   // "WT": the wait of vdit_wait_check ran out, as it should

// one warp waits for an arrival that nothing makes
__global__ void wait_check_kernel() {
    __shared__ uint64_t bar;
    __shared__ int abort_flag;
    if (threadIdx.x == 0) {
        tc::mbar_init(tc::smem_u32(&bar), 1);
        abort_flag = 0;
    }
    __syncthreads();
    tc::mbar_wait(tc::smem_u32(&bar), 0, &abort_flag, &g_wait_check_error, kErrWaitCheck);
}

}  // namespace

int wait_check_error_word(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_wait_check_error, sizeof(int)) != cudaSuccess) return VDIT_ERR_LAUNCH;
    if (clear) {
        int z = 0;
        if (cudaMemcpyToSymbol(g_wait_check_error, &z, sizeof(int)) != cudaSuccess) return VDIT_ERR_LAUNCH;
    }
    return v;
}

static std::atomic<long long> g_launches{0};

void count_launches(int n) { g_launches.fetch_add(n, std::memory_order_relaxed); }

static thread_local char g_last_error[256] = "";

void record_cuda_error(cudaError_t e) {
    snprintf(g_last_error, sizeof(g_last_error), "%s: %s", cudaGetErrorName(e), cudaGetErrorString(e));
}

}  // namespace vdit

extern "C" const char* vdit_last_cuda_error(void) { return vdit::g_last_error; }

extern "C" const char* vdit_version(void) { return "vdit 0.1 (sm_100a)"; }

extern "C" const char* vdit_error_string(int code) {
    switch (code) {
        case VDIT_OK: return "ok";
        case VDIT_ERR_ARG: return "invalid argument (shape, size or null pointer)";
        case VDIT_ERR_ALIGN: return "pointer or stride not 16-byte aligned";
        case VDIT_ERR_LAUNCH: return "CUDA launch failed";
        case VDIT_ERR_UNSUPPORTED: return "unsupported head_dim or width";
        case VDIT_ERR_WORKSPACE: return "workspace missing or too small";
        case VDIT_ERR_DRIVER: return "CUDA driver entry point failed";
        case VDIT_ERR_TOO_LARGE: return "size exceeds the fixed scratch of the no-alloc entry point";
        default: return "unknown error";
    }
}

extern "C" int vdit_wait_limit_ms(void) { return (int)(vdit::tc::kWaitLimitNs / 1000000u); }

extern "C" int vdit_wait_check(vdit_stream_t stream) {
    vdit::wait_check_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>();
    vdit::count_launches(1);
    return vdit::check_launch();
}

extern "C" long long vdit_launch_count(void) { return vdit::g_launches.load(std::memory_order_relaxed); }

