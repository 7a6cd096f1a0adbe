// Matrices to and from 4-bit microscaled floating point (mx.cuh): the operands of the
// block-scaled GEMM (mxlinear.cu).
//
// Both directions stream: rows x cols elements of 2 or 4 bytes on one side, 17 bytes per block of
// 32 on the other, so HBM bounds them.  A half warp takes 128 columns (four blocks, 8 elements a
// thread) of the four rows r, r + 32, r + 64, r + 96 of a 128-row block: its four 16-byte loads
// are independent, and the four rows' scale words are the 16 consecutive bytes of one scale
// block, so they leave (or arrive) as one vector.  The two half warps of a warp take
// neighbouring r, which makes the scale vector a whole 32-byte sector.
#include "mx.cuh"

namespace vdit {
namespace mx {
namespace {

constexpr int kThreads = 256;

// unit (half warp) -> row block, first row in it, 128-column group
struct Unit {
    int64_t rb;
    int r, g;
};
__device__ __forceinline__ Unit unit_of(int64_t u, int groups) {
    const int64_t pair = u >> 1;               // (row block, r / 2, group), group fastest
    const int64_t rest = pair / groups;
    return {rest >> 4, (int)(rest & 15) * 2 + (int)(u & 1), (int)(pair - rest * groups)};
}

template <int T>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const typename Elem<T>::type* __restrict__ x, int64_t ldx,
                                                            int64_t rows, int cols, int groups, int64_t units,
                                                            uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    asm volatile("griddepcontrol.launch_dependents;");      // a product of this matrix may set itself up meanwhile
    const int64_t u = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 4;
    if (u >= units) return;                    // whole half warps leave; the shuffles below stay in one
    const int l = threadIdx.x & 15;
    const unsigned half = 0xffffu << (threadIdx.x & 16);
    const Unit un = unit_of(u, groups);
    const int col = un.g * 128 + l * 8;
    const bool in_cols = col < cols;           // cols is a multiple of 32: a block is in or out as one
    float f[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = un.rb * 128 + un.r + 32 * i;
        if (in_cols && row < rows) {
            load8_f32(x + row * ldx + col, f[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
        }
    }
    uint32_t word[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = un.rb * 128 + un.r + 32 * i;
        uint32_t m = amax8(f[i]);
        m = max(m, __shfl_xor_sync(half, m, 1));
        m = max(m, __shfl_xor_sync(half, m, 2));
        const uint32_t s = scale_byte<4>(m);
        const float inv = scale_inverse(s);
        if (in_cols && row < rows) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = s == 255 ? 0.f : f[i][j] * inv;
            *reinterpret_cast<uint32_t*>(codes + row * (cols / 2) + col / 2) = encode8_e2m1(y);
        }
        uint32_t w = s << (8 * (l >> 2));      // this block's byte of the row's scale word
        w |= __shfl_xor_sync(half, w, 4);
        w |= __shfl_xor_sync(half, w, 8);
        word[i] = w;
    }
    if (l == 0)
        *reinterpret_cast<uint4*>(scales + (un.rb * groups + un.g) * 512 + un.r * 16) =
            make_uint4(word[0], word[1], word[2], word[3]);
}

template <int T>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales, int64_t rows,
                                                              int cols, int groups, int64_t units,
                                                              typename Elem<T>::type* __restrict__ out, int64_t ldo) {
    const int64_t u = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 4;
    if (u >= units) return;
    const int l = threadIdx.x & 15;
    const Unit un = unit_of(u, groups);
    const int col = un.g * 128 + l * 8;
    if (col >= cols) return;
    const uint4 sw = __ldg(reinterpret_cast<const uint4*>(scales + (un.rb * groups + un.g) * 512 + un.r * 16));
    const uint32_t word[4] = {sw.x, sw.y, sw.z, sw.w};
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = un.rb * 128 + un.r + 32 * i;
        c[i] = row < rows ? __ldg(reinterpret_cast<const uint32_t*>(codes + row * (cols / 2) + col / 2)) : 0u;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = un.rb * 128 + un.r + 32 * i;
        if (row >= rows) break;
        const float s = scale_value((word[i] >> (8 * (l >> 2))) & 255u);
        __half2 h[4];
        decode8_e2m1(c[i], h);
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 t = __half22float2(h[j]);
            f[2 * j] = t.x * s;
            f[2 * j + 1] = t.y * s;
        }
        store8_f32(out + row * ldo + col, f);
    }
}

// blocks of a launch over rows x cols, or 0 when they do not fit a grid
int64_t grid_of(int64_t rows, int cols, int64_t* units) {
    *units = scale_row_blocks(rows) * 32 * scale_col_groups(cols);
    const int64_t blocks = (*units * 16 + kThreads - 1) / kThreads;
    return blocks <= (int64_t)INT32_MAX ? blocks : 0;
}

// shape, stride and alignment checks shared by both directions (elem: bytes of a dense element)
int check_args(const void* dense, int64_t ld, int64_t rows, int32_t cols, int elem, const void* codes,
               const void* scales) {
    if (!dense || !codes || !scales || rows < 0 || cols <= 0 || ld < cols) return VDIT_ERR_ARG;
    if (cols % kBlock) return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(dense) || !aligned16(codes) || !aligned16(scales) || (ld * elem) % 16) return VDIT_ERR_ALIGN;
    return VDIT_OK;
}

int elem_bytes(int32_t type) { return type == VDIT_F32 ? 4 : type == VDIT_BF16 || type == VDIT_F16 ? 2 : 0; }

}  // namespace
}  // namespace mx
}  // namespace vdit

using namespace vdit;
using namespace vdit::mx;

extern "C" size_t vdit_mxfp4_scale_bytes(int64_t rows, int32_t cols) {
    if (rows < 0 || cols < 1) return 0;
    return (size_t)scale_row_blocks(rows) * scale_col_groups(cols) * 512;
}

extern "C" int vdit_mxfp4_quantize(const void* x, int32_t x_type, int64_t ldx, int64_t rows, int32_t cols,
                                   void* codes, void* scales, vdit_stream_t stream) {
    const int elem = elem_bytes(x_type);
    if (!elem) return VDIT_ERR_ARG;
    const int rc = check_args(x, ldx, rows, cols, elem, codes, scales);
    if (rc != VDIT_OK || rows == 0) return rc;
    int64_t units;
    const int64_t blocks = grid_of(rows, cols, &units);
    if (!blocks) return VDIT_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int groups = scale_col_groups(cols);
    auto run = [&](auto tag) {
        constexpr int T = decltype(tag)::value;
        quantize_kernel<T><<<(unsigned)blocks, kThreads, 0, s>>>(static_cast<const typename Elem<T>::type*>(x), ldx, rows,
                                                                cols, groups, units, static_cast<uint8_t*>(codes),
                                                                static_cast<uint8_t*>(scales));
    };
    if (x_type == VDIT_BF16) run(std::integral_constant<int, VDIT_BF16>{});
    else if (x_type == VDIT_F16) run(std::integral_constant<int, VDIT_F16>{});
    else run(std::integral_constant<int, VDIT_F32>{});
    count_launches(1);
    return check_launch();
}

extern "C" int vdit_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int32_t cols, void* out,
                                     int32_t out_type, int64_t ldo, vdit_stream_t stream) {
    const int elem = elem_bytes(out_type);
    if (!elem) return VDIT_ERR_ARG;
    const int rc = check_args(out, ldo, rows, cols, elem, codes, scales);
    if (rc != VDIT_OK || rows == 0) return rc;
    int64_t units;
    const int64_t blocks = grid_of(rows, cols, &units);
    if (!blocks) return VDIT_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int groups = scale_col_groups(cols);
    auto run = [&](auto tag) {
        constexpr int T = decltype(tag)::value;
        dequantize_kernel<T><<<(unsigned)blocks, kThreads, 0, s>>>(
            static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), rows, cols, groups, units,
            static_cast<typename Elem<T>::type*>(out), ldo);
    };
    if (out_type == VDIT_BF16) run(std::integral_constant<int, VDIT_BF16>{});
    else if (out_type == VDIT_F16) run(std::integral_constant<int, VDIT_F16>{});
    else run(std::integral_constant<int, VDIT_F32>{});
    count_launches(1);
    return check_launch();
}
