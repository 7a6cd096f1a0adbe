// Linear on 4-bit microscaled operands (mx.cuh):
//   out[m, n] = bf16( sum over blocks b of 2^(sa[m,b] + sw[n,b]) * sum_{j < 32} a[m,b,j] w[n,b,j] + bias[n] )
// Within a block the products are multiples of 1/4 below 1152 in sum, exact in fp32.
#include "mx.cuh"

namespace vdit {
namespace mx {
namespace {

constexpr int kTile = 64;

// 64 x 64 outputs a CTA, one block of 32 at a time through shared memory, 4 x 4 outputs a thread.
__global__ void __launch_bounds__(256) linear_tile_kernel(const uint8_t* __restrict__ a, const uint8_t* __restrict__ as,
                                                          const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
                                                          const __nv_bfloat16* __restrict__ bias,
                                                          __nv_bfloat16* __restrict__ out, int64_t ldo, int64_t m,
                                                          int n, int k) {
    __shared__ float sa[kBlock][kTile + 1], sw[kBlock][kTile + 1], ea[kTile], ew[kTile];
    const int64_t m0 = (int64_t)blockIdx.y * kTile;
    const int n0 = blockIdx.x * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int groups = scale_col_groups(k);
    float acc[4][4] = {};
    for (int b = 0; b < k / kBlock; ++b) {
        const int r = threadIdx.x >> 2, c = threadIdx.x & 3;       // row of the tile, 8 elements of its block
        const int64_t ra = m0 + r, rw = n0 + r;
        const uint32_t ca = ra < m ? *reinterpret_cast<const uint32_t*>(a + ra * (k / 2) + b * 16 + c * 4) : 0u;
        const uint32_t cw = rw < n ? *reinterpret_cast<const uint32_t*>(w + rw * (k / 2) + b * 16 + c * 4) : 0u;
        __half2 ha[4], hw[4];
        decode8_e2m1(ca, ha);
        decode8_e2m1(cw, hw);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 fa = __half22float2(ha[j]), fw = __half22float2(hw[j]);
            sa[c * 8 + 2 * j][r] = fa.x;
            sa[c * 8 + 2 * j + 1][r] = fa.y;
            sw[c * 8 + 2 * j][r] = fw.x;
            sw[c * 8 + 2 * j + 1][r] = fw.y;
        }
        if (threadIdx.x < 2 * kTile) {
            const int t = threadIdx.x & (kTile - 1);
            const bool is_a = threadIdx.x < kTile;
            const int64_t row = is_a ? m0 + t : n0 + t;
            const uint8_t* s = is_a ? as : ws;
            const bool in = row < (is_a ? m : (int64_t)n);
            (is_a ? ea : ew)[t] = in ? scale_value(s[((row >> 7) * groups + (b >> 2)) * 512 + (row & 31) * 16 +
                                                     ((row >> 5) & 3) * 4 + (b & 3)])
                                     : 0.f;
        }
        __syncthreads();
        float dot[4][4] = {};
#pragma unroll
        for (int j = 0; j < kBlock; ++j) {
            float va[4], vw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                va[i] = sa[j][ty + 16 * i];
                vw[i] = sw[j][tx + 16 * i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) dot[i][q] = fmaf(va[i], vw[q], dot[i][q]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][q] = fmaf(dot[i][q] * ea[ty + 16 * i], ew[tx + 16 * q], acc[i][q]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + ty + 16 * i;
        if (row >= m) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int col = n0 + tx + 16 * q;
            if (col < n) out[row * ldo + col] = f2bf(acc[i][q] + (bias ? bf2f(bias[col]) : 0.f));
        }
    }
}

}  // namespace
}  // namespace mx
}  // namespace vdit

using namespace vdit;
using namespace vdit::mx;

extern "C" int vdit_linear_mxfp4(const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales,
                                 const void* bias, void* out, int64_t ldo, int64_t m, int32_t n, int32_t k,
                                 vdit_stream_t stream) {
    if (!a_codes || !a_scales || !w_codes || !w_scales || !out || m < 0 || n <= 0 || k <= 0 || ldo < n)
        return VDIT_ERR_ARG;
    if (n % 8 || k % kBlock || m > (int64_t)INT32_MAX) return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(a_codes) || !aligned16(a_scales) || !aligned16(w_codes) || !aligned16(w_scales) || !aligned16(out) ||
        (bias && !aligned16(bias)) || ldo % 8)
        return VDIT_ERR_ALIGN;
    if (m == 0) return VDIT_OK;
    if ((m + kTile - 1) / kTile > 65535) return VDIT_ERR_UNSUPPORTED;
    const dim3 grid((n + kTile - 1) / kTile, (unsigned)((m + kTile - 1) / kTile));
    linear_tile_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(a_codes), static_cast<const uint8_t*>(a_scales), static_cast<const uint8_t*>(w_codes),
        static_cast<const uint8_t*>(w_scales), static_cast<const __nv_bfloat16*>(bias), static_cast<__nv_bfloat16*>(out),
        ldo, m, n, k);
    count_launches(1);
    return check_launch();
}
