// Linear on 4-bit microscaled operands (mx.cuh) on the block-scaled tcgen05 MMA:
//   out[m, n] = bf16( sum over blocks b of 2^(sa[m,b] + sw[n,b]) * sum_{j < 32} a[m,b,j] w[n,b,j] + bias[n] )
//
// A persistent CTA per SM walks 128 x BN output tiles.  A k-step is 256 elements (128 bytes) of
// 128 rows of a and BN rows of w, and their scales.  Warp roles:
//   warp 0      TMA producer: the codes as 128-byte-wide boxes (128-byte swizzle, K-major), the
//               scales as untiled copies of the 512-byte blocks they are stored in, all of a
//               k-step on one barrier of a ring
//   warp 1      MMA issuer: copies the k-step's scales from shared memory to TMEM (tcgen05.cp; each
//               ring stage has its own columns, free when the stage is), then up to four
//               128 x BN x 64 MMAs into one of two TMEM accumulators
//   warps 2..5  epilogue: bias, rounding and TMA stores of one accumulator while the MMAs of the
//               next tile fill the other
// 192 columns is the widest tile whose two accumulators leave TMEM room for the scales (2 x 192 +
// 4 stages x 24 of 512 columns); its tiles start on every other 64 rows of w, so an odd tile reads
// its scales from two columns further on.
//
// Every mbarrier wait is bounded; a wait that runs out records an error in g_mxlinear_error,
// raises the CTA abort flag and the CTA skips to its teardown (TMEM always freed).
#include <string.h>

#include <algorithm>
#include <atomic>

#include "mx.cuh"
#include "tc.cuh"

namespace vdit {

__device__ int g_mxlinear_error = 0;

namespace mx {
namespace {

using namespace tc;

constexpr int BM = 128;
constexpr int BK = 256;                 // elements of a k-step: 128 bytes of codes
constexpr int EPI_WARPS = 4;
constexpr int kThreads = (2 + EPI_WARPS) * 32;
constexpr int kErr = 0x4D58;            // "MX": a bounded wait of the linear ran out
constexpr int kScaleBlock = 512;        // 128 rows x 4 scales

template <int BN>
struct __align__(1024) Smem {
    static constexpr int NBLK = BN == 192 ? 2 : 1;          // 128-row scale blocks a tile of w touches
    static constexpr int NST = BN == 192 ? 4 : BN == 128 ? 5 : 6;
    uint8_t a[NST][BM * 128];
    uint8_t w[NST][BN * 128];
    uint8_t x[EPI_WARPS * 2 * 32 * 128];                    // two 32-row x 64-column boxes a warp
    uint8_t sa[NST][2 * kScaleBlock];
    uint8_t sw[NST][NBLK][2 * kScaleBlock];
    uint64_t full[NST], empty[NST], acc_full[2], acc_empty[2];
    uint32_t tmem_slot;
    int abort_flag;
};

struct Args {
    const uint8_t *as, *ws;             // scales
    const __nv_bfloat16* bias;
    int64_t m;
    int n, k;
};

// tile t -> (row tile, column tile): bands of 8 row tiles, so the rows in flight stay in L2 while
// the weight passes over them
__device__ __forceinline__ void tile_coords(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
    constexpr int GM = 8;
    const int g = t / (GM * tiles_n), within = t - g * GM * tiles_n;
    const int gm = min(GM, tiles_m - g * GM);
    tm = g * GM + within % gm;
    tn = within / gm;
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(y)
                 : "memory");
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1) linear_kernel(const __grid_constant__ CUtensorMap tmA,
                                                             const __grid_constant__ CUtensorMap tmW,
                                                             const __grid_constant__ CUtensorMap tmO,
                                                             const __grid_constant__ Args p) {
    extern __shared__ uint8_t raw[];
    using SM = Smem<BN>;
    constexpr int NST = SM::NST, NBLK = SM::NBLK;
    constexpr uint32_t kSfCols = 8 + 8 * NBLK;              // TMEM columns of one stage's scales
    constexpr uint32_t kTmemCols = 2 * BN + NST * kSfCols <= 256 ? 256 : 512;
    static_assert(2 * BN + NST * kSfCols <= 512, "TMEM");
    SM& sm = *reinterpret_cast<SM*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int* abort_flag = &sm.abort_flag;
    // rows, columns and steps past the operands read zeros (the tensor maps' fill); a k-step
    // runs only the MMAs that k reaches
    const int tiles_m = (int)((p.m + BM - 1) / BM), tiles_n = (p.n + BN - 1) / BN;
    const int ntiles = tiles_m * tiles_n;
    const int nk = (p.k + BK - 1) / BK;
    const int groups = scale_col_groups(p.k);

    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbar_init(smem_u32(&sm.full[s]), 1);
            mbar_init(smem_u32(&sm.empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&sm.acc_full[b]), 1);
            mbar_init(smem_u32(&sm.acc_empty[b]), EPI_WARPS);
        }
        sm.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmA)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmW)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmO)) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&sm.tmem_slot)), "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_slot;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            const int w_blocks = (p.n + 127) / 128;
            int it = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x) {
                int tm, tn;
                tile_coords(t, tiles_m, tiles_n, tm, tn);
                const int wb = tn * BN / 128;               // first scale block of the tile's rows of w
                const int nb = min(NBLK, w_blocks - wb);
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int s = it % NST;
                    if (it >= NST &&
                        !mbar_wait(smem_u32(&sm.empty[s]), ((it / NST) - 1) & 1, abort_flag, &g_mxlinear_error, kErr)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = smem_u32(&sm.full[s]);
                    const uint32_t sf = (uint32_t)min(2, groups - 2 * kb) * kScaleBlock;
                    mbar_expect_tx(bar, (BM + BN) * 128 + (1 + nb) * sf);
                    tma_load_2d(smem_u32(sm.a[s]), &tmA, kb * 128, tm * BM, bar);
                    tma_load_2d(smem_u32(sm.w[s]), &tmW, kb * 128, tn * BN, bar);
                    bulk_load(smem_u32(sm.sa[s]), p.as + ((int64_t)tm * groups + 2 * kb) * kScaleBlock, sf, bar);
                    for (int j = 0; j < nb; ++j)
                        bulk_load(smem_u32(sm.sw[s][j]), p.ws + ((int64_t)(wb + j) * groups + 2 * kb) * kScaleBlock, sf,
                                  bar);
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        // the whole warp runs the loop, the elected lane issues, with descriptors as bases plus
        // stage and k offsets so they stay in uniform registers
        const uint64_t ad0 = make_desc(smem_u32(sm.a[0]), 16, 1024, kSw128);
        const uint64_t wd0 = make_desc(smem_u32(sm.w[0]), 16, 1024, kSw128);
        const uint64_t sad0 = make_desc(smem_u32(sm.sa[0]), 16, 128, 0);
        const uint64_t swd0 = make_desc(smem_u32(sm.sw[0]), 16, 128, 0);
        auto wait = [&](uint32_t bar, uint32_t parity) {
            return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, &g_mxlinear_error, kErr));
        };
        int it = 0, lt = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < ntiles; t += gridDim.x, ++lt) {
            const int buf = lt & 1;
            int tm, tn;
            tile_coords(t, tiles_m, tiles_n, tm, tn);
            const uint32_t shift = (uint32_t)(tn * BN % 128) / 32;     // scale columns before the tile's first row
            if (lt >= 2 && !wait(smem_u32(&sm.acc_empty[buf]), ((lt >> 1) - 1) & 1)) break;
            tc_fence_after();
            const uint32_t acc = tmem + buf * BN;
            for (int kb = 0; kb < nk; ++kb, ++it) {
                const int s = it % NST;
                if (!wait(smem_u32(&sm.full[s]), (it / NST) & 1)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t ad = ad0 + (uint64_t)(s * (int)(sizeof(sm.a[0]) >> 4));
                const uint64_t wd = wd0 + (uint64_t)(s * (int)(sizeof(sm.w[0]) >> 4));
                const uint64_t sad = sad0 + (uint64_t)(s * (int)(sizeof(sm.sa[0]) >> 4));
                const uint64_t swd = swd0 + (uint64_t)(s * (int)(sizeof(sm.sw[0]) >> 4));
                const uint32_t sfa = tmem + 2 * BN + s * kSfCols, sfw = sfa + 8;
                const int ng = min(2, groups - 2 * kb), nm = min(4, (p.k - kb * BK + 63) / 64);
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    if (g < ng) {
                        tc_cp_scales_elect(sfa + 4 * g, sad + (uint64_t)(g * (kScaleBlock >> 4)));
#pragma unroll
                        for (int j = 0; j < NBLK; ++j)
                            tc_cp_scales_elect(sfw + 4 * (g * NBLK + j),
                                               swd + (uint64_t)((j * 2 + g) * (kScaleBlock >> 4)));
                    }
                }
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    if (kk < nm)
                        tc_mma_mxf4_elect(acc, ad + (uint64_t)(kk * 2), wd + (uint64_t)(kk * 2),
                                          make_idesc_mxf4(BM, BN, (kk & 1) * 2), sfa + 4 * (kk >> 1),
                                          sfw + 4 * NBLK * (kk >> 1) + shift, (kb > 0 || kk > 0) ? 1u : 0u);
                tc_commit_elect(smem_u32(&sm.empty[s]));
            }
            if (ok) tc_commit_elect(smem_u32(&sm.acc_full[buf]));
        }
    } else {
        // ------------------------------------------------------------ epilogue
        // Each warp turns 64 columns of its 32 rows at a time into bf16 in one of its two staging
        // boxes (128-byte swizzle) and one lane stores the box; the map clips rows past m and
        // columns past n.
        const int ew = warp - 2, quarter = warp & 3;
        const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
        int lt = 0, nstore = 0;
        for (int t = blockIdx.x; t < ntiles; t += gridDim.x, ++lt) {
            const int buf = lt & 1;
            int tm, tn;
            tile_coords(t, tiles_m, tiles_n, tm, tn);
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.acc_full[buf]), (lt >> 1) & 1, abort_flag,
                                                   &g_mxlinear_error, kErr)))
                break;
            tc_fence_after();
            const int64_t row0 = (int64_t)tm * BM + quarter * 32;
            const int col0 = tn * BN;
            if (row0 < p.m) {
#pragma unroll 1
                for (int c = 0; c < BN / 64; ++c) {
                    if (col0 + c * 64 >= p.n) break;
                    float v[64];
                    tmem_ld32(tmem + buf * BN + c * 64 + lane_off, v);
                    tmem_ld32(tmem + buf * BN + c * 64 + 32 + lane_off, v + 32);
                    tmem_wait_ld();
                    if (p.bias) {
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const int cb = col0 + c * 64 + q * 8;   // n is a multiple of 8
                            if (cb < p.n) {
                                float bv[8];
                                load8_nc(p.bias + cb, bv);
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[q * 8 + j] += bv[j];
                            }
                        }
                    }
                    uint8_t* box = sm.x + (ew * 2 + (nstore & 1)) * 32 * 128;
                    ++nstore;
                    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        *reinterpret_cast<uint4*>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) = pack8(v + q * 8);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmO, smem_u32(box), col0 + c * 64, (int)row0);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.acc_empty[buf]));
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

bool make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t rows, int cols, int64_t ld_bytes,
              int box_rows, int box_cols) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld_bytes};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    cuuint32_t es[2] = {1, 1};
    return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxDevices = 64;

// the current device and its SM count (148 if it cannot be asked)
int current_device(int* sms) {
    int dev = 0;
    *sms = 148;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -1;
    if (cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) *sms = 148;
    return dev;
}

template <int BN>
int launch(const CUtensorMap& ma, const CUtensorMap& mo, const void* w, const Args& p, int dev, int sms,
           cudaStream_t s) {
    static std::atomic<bool> ready[kMaxDevices];            // the kernel's shared memory size is set, per device
    constexpr int smem = (int)sizeof(Smem<BN>) + 1024;
    if (!ready[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(linear_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) {
            record_cuda_error(e);
            return VDIT_ERR_LAUNCH;
        }
        ready[dev].store(true, std::memory_order_release);
    }
    CUtensorMap mw;
    if (!make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, p.n, p.k / 2, p.k / 2, BN, 128)) return VDIT_ERR_DRIVER;
    const int64_t tiles = ((p.m + BM - 1) / BM) * ((p.n + BN - 1) / BN);
    if (tiles > INT32_MAX - 1024) return VDIT_ERR_UNSUPPORTED;
    linear_kernel<BN><<<(unsigned)std::min<int64_t>(tiles, sms), kThreads, smem, s>>>(ma, mw, mo, p);
    count_launches(1);
    return check_launch();
}

// Tile width: 192 columns, or narrower ones when 192-column tiles would leave SMs idle and the
// narrower fill more of them (few rows: the weight is then read by more SMs).
int pick_bn(int64_t m, int n, int sms) {
    const int64_t tiles_m = (m + BM - 1) / BM;
    for (int bn : {192, 128})
        if (tiles_m * ((n + bn - 1) / bn) >= sms) return bn;
    return 64;
}

}  // namespace
}  // namespace mx

int mxlinear_error_word(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_mxlinear_error, sizeof(int)) != cudaSuccess) return VDIT_ERR_LAUNCH;
    if (clear) {
        int z = 0;
        if (cudaMemcpyToSymbol(g_mxlinear_error, &z, sizeof(int)) != cudaSuccess) return VDIT_ERR_LAUNCH;
    }
    return v;
}

}  // namespace vdit

using namespace vdit;
using namespace vdit::mx;

extern "C" int vdit_linear_mxfp4(const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales,
                                 const void* bias, void* out, int64_t ldo, int64_t m, int32_t n, int32_t k,
                                 vdit_stream_t stream) {
    if (!a_codes || !a_scales || !w_codes || !w_scales || !out || m < 0 || n <= 0 || k <= 0 || ldo < n)
        return VDIT_ERR_ARG;
    if (n % 8 || k % kBlock || m > (int64_t)INT32_MAX - BM) return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(a_codes) || !aligned16(a_scales) || !aligned16(w_codes) || !aligned16(w_scales) || !aligned16(out) ||
        (bias && !aligned16(bias)) || ldo % 8)
        return VDIT_ERR_ALIGN;
    if (m == 0) return VDIT_OK;
    int sms;
    const int dev = current_device(&sms);
    if (dev < 0) return VDIT_ERR_UNSUPPORTED;
    CUtensorMap ma, mo;
    if (!make_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, a_codes, m, k / 2, k / 2, BM, 128) ||
        !make_map(&mo, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, out, m, n, ldo * 2, 32, 64))
        return VDIT_ERR_DRIVER;
    const Args p{static_cast<const uint8_t*>(a_scales), static_cast<const uint8_t*>(w_scales),
                 static_cast<const __nv_bfloat16*>(bias), m, n, k};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (pick_bn(m, n, sms)) {
        case 192: return launch<192>(ma, mo, w_codes, p, dev, sms, s);
        case 128: return launch<128>(ma, mo, w_codes, p, dev, sms, s);
        default: return launch<64>(ma, mo, w_codes, p, dev, sms, s);
    }
}
