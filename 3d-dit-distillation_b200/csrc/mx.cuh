// Microscaled (MX) number formats: blocks of 32 consecutive elements of a row share one
// power-of-two scale byte s (ue8m0: 2^(s - 127), 255 = NaN), elements are e2m1 (4 bits,
// +-{0, .5, 1, 1.5, 2, 3, 4, 6}) or e4m3 (8 bits, up to 448).
//
// Quantising a block x: s - 127 = floor(log2(max|x|)) - emax, emax the exponent of the element
// type's largest value (2 for e2m1, 8 for e4m3), no lower than -127; element = x * 2^(127 - s)
// rounded to the nearest element value (ties to even, no further than the largest).  The scaling
// is exact, so the one rounding is the element's.  A block with a NaN or an infinity, which
// neither the 4-bit type nor the scale rule can hold, gets s = 255 and reads back as NaN.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace vdit {
namespace mx {

constexpr int kBlock = 32;

// element types of the matrices that are quantised or read back (vdit.h VDIT_BF16 ...)
template <int T> struct Elem;
template <> struct Elem<VDIT_BF16> { using type = __nv_bfloat16; };
template <> struct Elem<VDIT_F16> { using type = __half; };
template <> struct Elem<VDIT_F32> { using type = float; };

__device__ __forceinline__ float2 fmul2(float2 a, float s) {
    unsigned long long ra, rs, rd;
    asm("mov.b64 %0, {%1,%2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1,%1};" : "=l"(rs) : "f"(s));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rs));
    float2 o;
    asm("mov.b64 {%0,%1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(rd));
    return o;
}

__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
    unsigned long long ra, rb, rd;
    asm("mov.b64 %0, {%1,%2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1,%2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    float2 o;
    asm("mov.b64 {%0,%1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(rd));
    return o;
}

// Waits until the kernels before this one in the stream are complete and what they wrote is visible,
// then lets the next one set itself up.  In this order: when the next kernel starts, only this one is
// still running, so that neither waits pile up nor a bounded wait there counts an older kernel's time.
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Loads of what an earlier kernel may have written while this one was already there: not read-only for
// this kernel's whole life, so not through the read-only path (__ldg), and never moved above the wait.
__device__ __forceinline__ uint4 load_after(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint2 load_after(const uint2* p) {
    uint2 v;
    asm volatile("ld.global.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_after(const float4* p) {
    float4 v;
    asm volatile("ld.global.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ int64_t load_after(const int64_t* p) {
    int64_t v;
    asm volatile("ld.global.b64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ int32_t load_after(const int32_t* p) {
    int32_t v;
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t load_after(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// 16 consecutive elements (half a block) of a row as they are stored, their largest magnitude and
// their values.  The 16-bit types' magnitudes are compared two at a time as integers.
template <int T>
struct Half {
    uint4 u[2];
    __device__ __forceinline__ void load(const void* p) {
        u[0] = load_after(static_cast<const uint4*>(p));
        u[1] = load_after(static_cast<const uint4*>(p) + 1);
    }
    __device__ __forceinline__ void zero() { u[0] = u[1] = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4& q = u[i >> 2];
        return (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
    }
    __device__ __forceinline__ uint32_t amax() const {         // as fp32 bits
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = __vmaxu2(m, word(i) & 0x7fff7fffu);
        m = max(m >> 16, m & 0xffffu);
        return T == VDIT_BF16 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    }
    __device__ __forceinline__ float2 pair(int i) const {
        const uint32_t w = word(i);
        if (T == VDIT_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    }
};
template <>
struct Half<VDIT_F32> {
    float4 u[4];
    __device__ __forceinline__ void load(const void* p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = load_after(static_cast<const float4*>(p) + i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __device__ __forceinline__ float2 pair(int i) const {
        const float4& q = u[i >> 1];
        return i & 1 ? make_float2(q.z, q.w) : make_float2(q.x, q.y);
    }
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 v = pair(i);
            m = max(m, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
        }
        return m;
    }
};

// max |f[i]| as fp32 bits: as integers the magnitudes order like the numbers, with the
// infinity above every finite value and the NaNs above the infinity, so nothing is dropped
__device__ __forceinline__ uint32_t amax8(const float* f) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    return m;
}

// the scale byte of a block from its max |x| (fp32 bits).  The exponent field of a subnormal is
// 0: below 2^-126 every block has the smallest scale.
template <int BITS>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
    constexpr int emax = BITS == 4 ? 2 : 8;
    const int e = (int)(amax >> 23);
    return e == 255 ? 255u : (uint32_t)max(e - emax, 0);
}

// 2^(s - 127); s = 0 is the subnormal 2^-127, s = 255 a NaN
__device__ __forceinline__ float scale_value(uint32_t s) {
    return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fffffffu : s << 23);
}
// 2^(127 - s) for a scale of scale_byte (s <= 252), 0 for a NaN block (all its codes 0)
__device__ __forceinline__ float scale_inverse(uint32_t s) {
    return s == 255 ? 0.f : __uint_as_float((254u - s) << 23);
}

// 8 elements (already scaled) to codes: BITS bytes, element 0 in the lowest bits
__device__ __forceinline__ uint32_t encode8_e2m1(const float* f) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return r;
}
__device__ __forceinline__ uint2 encode8_e4m3(const float* f) {
    uint2 r;
    asm("{\n\t.reg .b16 h0, h1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h0, %3, %2;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h1, %5, %4;\n\t"
        "mov.b32 %0, {h0, h1};\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h0, %7, %6;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h1, %9, %8;\n\t"
        "mov.b32 %1, {h0, h1};\n\t}"
        : "=r"(r.x), "=r"(r.y)
        : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return r;
}

// the e2m1 value nearest to y, ties to even, no further than 6, in fp32: adding and taking away
// 1.5 * 2^23 units rounds to a unit, half below 2, one below 4, two above.  (Where the codes are not
// stored: encode8_e2m1 and decode8_e2m1 of its result in one kernel gave zeros, compiled by nvcc 12.9.)
__device__ __forceinline__ float round_e2m1(float y) {
    const float a = fabsf(y), big = a < 2.f ? 6291456.f : a < 4.f ? 12582912.f : 25165824.f;
    return copysignf(fminf((a + big) - big, 6.f), y);
}

// Stores half a block's 16 values of this lane (even: the first, odd: the second half of a block that
// the lanes 2i and 2i + 1 hold; both call).  Each lane's 16-byte pieces lie 32 bytes apart from its
// neighbour's, so the two swap pieces first and every store of the warp is one consecutive run
// (38 -> 30 us for 16384 x 3840 bf16).  `out`: this lane's 16 elements.
__device__ __forceinline__ uint4 swap_piece(uint4 mine) {
    const unsigned pair = 3u << (threadIdx.x & 30);
    return make_uint4(__shfl_xor_sync(pair, mine.x, 1), __shfl_xor_sync(pair, mine.y, 1),
                      __shfl_xor_sync(pair, mine.z, 1), __shfl_xor_sync(pair, mine.w, 1));
}
// PIECES consecutive 16-byte pieces a lane, an even number
template <int PIECES>
__device__ __forceinline__ void store_pieces(uint4* out, uint4 (&v)[PIECES]) {
    // lane-pair transpose of 2 x 2 pieces at a time: pieces (2j, 2j + 1) of both lanes
    const bool odd = threadIdx.x & 1;
#pragma unroll
    for (int j = 0; j < PIECES; j += 2) {
        const uint4 got = swap_piece(odd ? v[j] : v[j + 1]);
        // even: own piece j and the odd lane's piece j; odd: the even lane's piece j + 1 and its own
        const uint4 a = odd ? got : v[j], b = odd ? v[j + 1] : got;
        uint4* base = out + j + (odd ? 1 - PIECES : 0);
        base[0] = a;
        base[PIECES] = b;
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename E>
__device__ __forceinline__ void store_half(E* out, const float* f) {
    uint4 v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        v[i] = make_uint4(pack2(f[8 * i], f[8 * i + 1], E{}), pack2(f[8 * i + 2], f[8 * i + 3], E{}),
                          pack2(f[8 * i + 4], f[8 * i + 5], E{}), pack2(f[8 * i + 6], f[8 * i + 7], E{}));
    store_pieces(reinterpret_cast<uint4*>(out), v);
}
__device__ __forceinline__ void store_half(float* out, const float* f) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                          __float_as_uint(f[4 * i + 3]));
    store_pieces(reinterpret_cast<uint4*>(out), v);
}

// half a block's codes, BITS * 2 bytes; 0 in a block without a scale
template <int T>
__device__ __forceinline__ uint2 encode_half_e2m1(const Half<T>& x, uint32_t s) {
    const float inv = scale_inverse(s);
    float f[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 y = fmul2(x.pair(i), inv);
        f[2 * i] = y.x;
        f[2 * i + 1] = y.y;
    }
    return s == 255 ? make_uint2(0, 0) : make_uint2(encode8_e2m1(f), encode8_e2m1(f + 8));
}
template <int T>
__device__ __forceinline__ uint4 encode_half_e4m3(const Half<T>& x, uint32_t s) {
    const float inv = scale_inverse(s);
    float f[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 y = fmul2(x.pair(i), inv);
        f[2 * i] = y.x;
        f[2 * i + 1] = y.y;
    }
    const uint2 a = encode8_e4m3(f), b = encode8_e4m3(f + 8);
    return s == 255 ? make_uint4(0, 0, 0, 0) : make_uint4(a.x, a.y, b.x, b.y);
}

// codes to f16 pairs (every element value is an f16 value)
__device__ __forceinline__ void decode8_e2m1(uint32_t c, __half2* h) {
    uint32_t r[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
        : "r"(c));
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<__half2*>(&r[i]);
}
__device__ __forceinline__ void decode4_e4m3(uint32_t c, __half2* h) {
    uint32_t r[2];
    asm("{\n\t.reg .b16 h0, h1;\n\t"
        "mov.b32 {h0, h1}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, h0;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h1;\n\t}"
        : "=r"(r[0]), "=r"(r[1])
        : "r"(c));
#pragma unroll
    for (int i = 0; i < 2; ++i) h[i] = *reinterpret_cast<__half2*>(&r[i]);
}

// A launch that may be set up while the kernel before it in the stream ends; the kernel calls
// after_previous() in every thread before it touches global memory.
// It saves the gap between two calls of a stream, 1.5 to 2 us a launch (quantise and read back 7680 x 1536:
// 26.4 -> 21.5 us; write and read back 4101 rows of 12 x 128: 21.5 -> 17.2), not time of the kernels.
template <typename... Params, typename... Args>
inline cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, cudaStream_t s, Args... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
    if (e != cudaSuccess) record_cuda_error(e);             // check_launch() then reports it, too
    return e;
}

// The scales of a quantised matrix [rows, cols] are held in the order the block-scaled MMA
// takes them from shared memory: 128 rows x 4 scales (128 columns) make one 512-byte block,
// scale j of row r at (r % 32) * 16 + (r / 32) * 4 + j; the blocks of 128 rows follow one
// another along the columns.  Rows and scales past the matrix are 0.
__host__ __device__ constexpr int64_t scale_row_blocks(int64_t rows) { return (rows + 127) / 128; }
__host__ __device__ constexpr int scale_col_groups(int cols) { return (cols + 127) / 128; }

}  // namespace mx
}  // namespace vdit
