// Matrices to and from 4-bit microscaled floating point (mx.cuh): the operands of the
// block-scaled GEMM (mxlinear.cu).
//
// Both directions stream: rows x cols elements of 2 or 4 bytes on one side, 17 bytes per block of
// 32 on the other, so HBM bounds them once the instructions an element takes are few: a thread takes
// half a block at a time (16.7 instructions an element with a quarter block, 64-bit divisions for the
// position and fp32 magnitudes: 42 us for 16384 x 3840 bf16, against 28 us).  Eight threads take
// 128 columns (four blocks) of the four rows r, r + 32, r + 64, r + 96 of a 128-row block: their
// loads are independent, and the four rows' scale words are the 16 consecutive bytes of one scale
// block, so they leave (or arrive) as one vector.  A warp takes four neighbouring r, a CTA eight
// groups of 128 columns of them.
#include "mx.cuh"

namespace vdit {
namespace mx {
namespace {

constexpr int kThreads = 256;

// blockIdx.x: 128-row block and four rows r of its first 32; blockIdx.y and the warp: group of 128 columns
struct Place {
    int64_t row;      // r; the thread's rows are row + 32 i
    int col;
    int64_t scale;    // byte of the scale vector
};
__device__ __forceinline__ Place place_of(int groups, int* group) {
    const int g = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int64_t rb = blockIdx.x >> 3;
    const int r = (blockIdx.x & 7) * 4 + (lane >> 3);
    *group = g;
    return {rb * 128 + r, g * 128 + (lane & 7) * 16, (rb * groups + g) * 512 + r * 16};
}

template <int T>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const typename Elem<T>::type* x, int64_t ldx,
                                                            int64_t rows, int cols, int groups,
                                                            uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    after_previous();                                       // a product of this matrix may then set itself up
    int g;
    const Place at = place_of(groups, &g);
    if (g >= groups) return;                                // whole warps leave
    const int part = threadIdx.x & 7;
    const bool in_cols = at.col < cols;                     // cols is a multiple of 32: a block is in or out as one
    Half<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (in_cols && at.row + 32 * i < rows) v[i].load(x + (at.row + 32 * i) * ldx + at.col);
        else v[i].zero();
    }
    uint32_t word[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t m = v[i].amax();
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const uint32_t s = scale_byte<4>(m);
        if (in_cols && at.row + 32 * i < rows)
            *reinterpret_cast<uint2*>(codes + (at.row + 32 * i) * (cols / 2) + at.col / 2) = encode_half_e2m1(v[i], s);
        uint32_t w = s << (8 * (part >> 1));                // this block's byte of the row's scale word
        w |= __shfl_xor_sync(0xffffffffu, w, 2);
        word[i] = w | __shfl_xor_sync(0xffffffffu, w, 4);
    }
    if (part == 0) *reinterpret_cast<uint4*>(scales + at.scale) = make_uint4(word[0], word[1], word[2], word[3]);
}

template <int T>
__global__ void __launch_bounds__(kThreads) dequantize_kernel(const uint8_t* codes,
                                                              const uint8_t* scales, int64_t rows,
                                                              int cols, int groups,
                                                              typename Elem<T>::type* __restrict__ out, int64_t ldo) {
    after_previous();
    int g;
    const Place at = place_of(groups, &g);
    if (g >= groups || at.col >= cols) return;
    const uint4 sw = load_after(reinterpret_cast<const uint4*>(scales + at.scale));
    const uint32_t word[4] = {sw.x, sw.y, sw.z, sw.w};
    uint2 c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        c[i] = at.row + 32 * i < rows
                   ? load_after(reinterpret_cast<const uint2*>(codes + (at.row + 32 * i) * (cols / 2) + at.col / 2))
                   : make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (at.row + 32 * i >= rows) break;
        const float s = scale_value((word[i] >> (8 * (threadIdx.x >> 1 & 3))) & 255u);
        __half2 h[8];
        decode8_e2m1(c[i].x, h);
        decode8_e2m1(c[i].y, h + 4);
        float f[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 t = fmul2(__half22float2(h[j]), s);
            f[2 * j] = t.x;
            f[2 * j + 1] = t.y;
        }
        store_half(out + (at.row + 32 * i) * ldo + at.col, f);
    }
}

// grid of a launch over rows x cols; x = 0 when it does not fit
dim3 grid_of(int64_t rows, int cols) {
    const int64_t x = scale_row_blocks(rows) * 8, y = (scale_col_groups(cols) + 7) / 8;
    return x > (int64_t)INT32_MAX || y > 65535 ? dim3(0, 0) : dim3((unsigned)x, (unsigned)y);
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
    const dim3 grid = grid_of(rows, cols);
    if (!grid.x) return VDIT_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int groups = scale_col_groups(cols);
    auto run = [&](auto tag) {
        constexpr int T = decltype(tag)::value;
        launch_early(quantize_kernel<T>, grid, kThreads, s, static_cast<const typename Elem<T>::type*>(x), ldx, rows, cols,
                     groups, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
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
    const dim3 grid = grid_of(rows, cols);
    if (!grid.x) return VDIT_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int groups = scale_col_groups(cols);
    auto run = [&](auto tag) {
        constexpr int T = decltype(tag)::value;
        launch_early(dequantize_kernel<T>, grid, kThreads, s, static_cast<const uint8_t*>(codes),
                     static_cast<const uint8_t*>(scales), rows, cols, groups,
                     static_cast<typename Elem<T>::type*>(out), ldo);
    };
    if (out_type == VDIT_BF16) run(std::integral_constant<int, VDIT_BF16>{});
    else if (out_type == VDIT_F16) run(std::integral_constant<int, VDIT_F16>{});
    else run(std::integral_constant<int, VDIT_F32>{});
    count_launches(1);
    return check_launch();
}
