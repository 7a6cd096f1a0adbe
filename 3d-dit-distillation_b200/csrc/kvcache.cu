// A paged key/value cache in microscaled 8- or 4-bit floating point (mx.cuh): written as rows
// arrive, read back as rows, and attended to by one query per sequence and head.
//
// Layout: slot = page * page_size + offset.  Keys (and, apart, values) are
// [pages, heads, page_size, head_dim * bits / 8] bytes and their scales
// [pages, heads, page_size, head_dim / 32] bytes, so the keys of one head in one page are
// consecutive: what one query head reads.
#include <math.h>

#include <atomic>

#include "mx.cuh"
#include "tc.cuh"

namespace vdit {

__device__ int g_kvcache_error = 0;

namespace kv {
namespace {

using namespace mx;

constexpr int kErrIndex = 0x4B56;   // "KV": a slot, page or length outside the cache
constexpr int kThreads = 256;
constexpr int kMaxSplits = 1024;

struct Cache {
    uint8_t *k, *v, *ks, *vs;
    int64_t pages;
    int page_size, page_shift, heads, hd;
};

// byte offsets of (slot, head)'s data and scales
template <int BITS>
__device__ __forceinline__ int64_t data_at(const Cache& c, int64_t page, int h, int off) {
    return ((page * c.heads + h) * c.page_size + off) * (int64_t)(c.hd * BITS / 8);
}
__device__ __forceinline__ int64_t scale_at(const Cache& c, int64_t page, int h, int off) {
    return ((page * c.heads + h) * c.page_size + off) * (int64_t)(c.hd / kBlock);
}

// ------------------------------------------------------------------ write and read back
// Streams: a thread takes 8 channels of one row's key and value (four neighbouring threads one
// block of 32), so a row's channels are read and its codes written by consecutive threads.
template <int BITS>
__device__ __forceinline__ void put8(const float* f, uint8_t* data, uint8_t* scale, bool first) {
    uint32_t m = amax8(f);
    const unsigned quad = 0xfu << (threadIdx.x & 28);
    m = max(m, __shfl_xor_sync(quad, m, 1));
    m = max(m, __shfl_xor_sync(quad, m, 2));
    const uint32_t s = scale_byte<BITS>(m);
    const float inv = scale_inverse(s);
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = s == 255 ? 0.f : f[j] * inv;
    if (BITS == 4) *reinterpret_cast<uint32_t*>(data) = encode8_e2m1(y);
    else *reinterpret_cast<uint2*>(data) = encode8_e4m3(y);
    if (first) *scale = (uint8_t)s;
}

template <int BITS>
__global__ void __launch_bounds__(kThreads) write_kernel(const __nv_bfloat16* __restrict__ k, int64_t ldk,
                                                         const __nv_bfloat16* __restrict__ v, int64_t ldv,
                                                         const int64_t* __restrict__ slots, int64_t n, Cache c) {
    const int per_row = c.heads * c.hd / 8;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = i / per_row;
    if (row >= n) return;
    const int ch = (int)(i - row * per_row) * 8;
    const int64_t slot = __ldg(slots + row);
    if (slot < 0) return;                                   // the four threads of a block agree
    if (slot >= c.pages * c.page_size) {
        atomicExch(&g_kvcache_error, kErrIndex);
        return;
    }
    const int h = ch / c.hd, e = ch - h * c.hd;
    const int64_t page = slot >> c.page_shift;
    const int off = (int)(slot & (c.page_size - 1));
    float fk[8], fv[8];
    load8_f32(k + row * ldk + ch, fk);
    load8_f32(v + row * ldv + ch, fv);
    const int64_t d = data_at<BITS>(c, page, h, off) + e * BITS / 8, s = scale_at(c, page, h, off) + e / kBlock;
    const bool first = (e & 31) == 0;
    put8<BITS>(fk, c.k + d, c.ks + s, first);
    put8<BITS>(fv, c.v + d, c.vs + s, first);
}

template <int BITS, typename T>
__device__ __forceinline__ void get8(const uint8_t* data, const uint8_t* scale, T* out) {
    const float s = scale_value(*scale);
    __half2 h[4];
    if (BITS == 4) {
        decode8_e2m1(*reinterpret_cast<const uint32_t*>(data), h);
    } else {
        const uint2 u = *reinterpret_cast<const uint2*>(data);
        decode4_e4m3(u.x, h);
        decode4_e4m3(u.y, h + 2);
    }
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 t = __half22float2(h[j]);
        f[2 * j] = t.x * s;
        f[2 * j + 1] = t.y * s;
    }
    store8_f32(out, f);
}

template <int BITS, typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(Cache c, const int64_t* __restrict__ slots, int64_t n,
                                                        T* __restrict__ k, int64_t ldk, T* __restrict__ v,
                                                        int64_t ldv) {
    const int per_row = c.heads * c.hd / 8;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = i / per_row;
    if (row >= n) return;
    const int ch = (int)(i - row * per_row) * 8;
    const int64_t slot = __ldg(slots + row);
    const bool outside = slot >= c.pages * c.page_size;
    if (outside) atomicExch(&g_kvcache_error, kErrIndex);
    if (slot < 0 || outside) {                              // no such row: zeros
        const float z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        store8_f32(k + row * ldk + ch, z);
        store8_f32(v + row * ldv + ch, z);
        return;
    }
    const int h = ch / c.hd, e = ch - h * c.hd;
    const int64_t page = slot >> c.page_shift;
    const int off = (int)(slot & (c.page_size - 1));
    const int64_t d = data_at<BITS>(c, page, h, off) + e * BITS / 8, s = scale_at(c, page, h, off) + e / kBlock;
    get8<BITS>(c.k + d, c.ks + s, k + row * ldk + ch);
    get8<BITS>(c.v + d, c.vs + s, v + row * ldv + ch);
}

// ------------------------------------------------------------------ single-query attention
// One query per sequence and head over the cached keys of the sequence's pages: a stream of
// head_dim * bits / 8 + head_dim / 32 bytes a key, twice, bound by HBM once the arithmetic keeps up.
// In fp32 on the CUDA cores it did not (an unpack, a conversion and an FMA an element and query: 312 us
// for 16 sequences of up to 32768 keys, 12 x 128 heads, 8 bits; 53 us for 16 of up to 6082 with four
// queries a key head), so both products run on mma.sync m16n8k16: a pair of elements is one
// conversion to f16 (exact for both element types) and up to 8 queries of a key head share it.
//
// A CTA takes one sequence, one key head, up to 8 of its queries and one range ("split") of the keys.
// Its warps are independent until the end: each takes every fourth group of 16 consecutive keys
// (they lie in one page), copied by cp.async into the warp's own ring, rows padded to an odd number
// of 16-byte chunks so that the fragment reads spread over the banks.  Per group and 32-channel block:
//   S = K Q^T   16 keys x 8 queries, times each key's scale in fp32.  Q is f16 after scaling each
//               query by a power of two that puts its largest channel at 2^13: exact but for
//               channels 2^27 below that one
//   O += V^T P  channels x queries, P = 2^(s - m) in f16 (a weight is off by 2^-12 of itself, an
//               eighth of the output's own rounding), each key's weight times its value scale
//               relative to the group's largest, which multiplies the product in fp32
// Channels and keys map to fragment indices so that a lane reads consecutive bytes.  m is raised
// only by a score more than 1 above it (the weights stay below 2, the f16 ones, times 2^14, below
// 2^15): exact, as every term uses the same m.
constexpr int kWarps = 4;
constexpr int kStages = 3;                   // groups of a warp in its ring
constexpr int kQ = 8;                        // queries of a CTA
constexpr int kGroup = 16;                   // keys of a group

struct AttnArgs {
    const __nv_bfloat16* q;
    int64_t ldq;
    __nv_bfloat16* out;
    int64_t ldo;
    const int32_t* table;                    // [batch, ldt] pages of each sequence
    int64_t ldt;
    const int32_t* lengths;                  // [batch]
    int max_pages;                           // entries of a table row
    int heads, group;                        // query heads, and how many share a key head
    int splits;
    float scale_log2;
    float* ws;                               // [batch, heads, splits, 2 + hd] when splits > 1
};

// a sequence's length, held inside its table row
__device__ __forceinline__ int64_t length_of(const AttnArgs& a, int page_size, int b) {
    const int64_t most = (int64_t)a.max_pages * page_size, n = __ldg(a.lengths + b);
    if (n < 0 || n > most) {
        atomicExch(&g_kvcache_error, kErrIndex);
        return n < 0 ? 0 : most;
    }
    return n;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// an 8 x 8 matrix of 16-bit elements, two of a row a lane, to its transpose
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 8 consecutive channels of a key to 4 f16 pairs
template <int BITS>
__device__ __forceinline__ void key_pairs(const uint8_t* p, uint32_t* h) {
    if (BITS == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        decode4_e4m3(u.x, reinterpret_cast<__half2*>(h));
        decode4_e4m3(u.y, reinterpret_cast<__half2*>(h) + 2);
    } else {
        decode8_e2m1(*reinterpret_cast<const uint32_t*>(p), reinterpret_cast<__half2*>(h));
    }
}

// 4 consecutive channels of two keys' values to f16 pairs (first key, second key) of each channel
template <int BITS>
__device__ __forceinline__ void value_pairs(const uint8_t* p0, const uint8_t* p1, uint32_t* h) {
    if (BITS == 8) {
        const uint32_t a = *reinterpret_cast<const uint32_t*>(p0), b = *reinterpret_cast<const uint32_t*>(p1);
        decode4_e4m3(__byte_perm(a, b, 0x5140), reinterpret_cast<__half2*>(h));
        decode4_e4m3(__byte_perm(a, b, 0x7362), reinterpret_cast<__half2*>(h) + 2);
    } else {
        const uint32_t a = *reinterpret_cast<const uint16_t*>(p0), b = *reinterpret_cast<const uint16_t*>(p1);
        // bytes: channels 0, 2 of both keys, then 1, 3
        const uint32_t even = (a & 0x0f0fu) | ((b << 4) & 0xf0f0u), od = ((a >> 4) & 0x0f0fu) | (b & 0xf0f0u);
        __half2 t[4];
        decode8_e2m1(even | (od << 16), t);
        h[0] = *reinterpret_cast<uint32_t*>(&t[0]);
        h[2] = *reinterpret_cast<uint32_t*>(&t[1]);
        h[1] = *reinterpret_cast<uint32_t*>(&t[2]);
        h[3] = *reinterpret_cast<uint32_t*>(&t[3]);
    }
}

// shared memory of a warp's ring and of the whole CTA
template <int HD, int BITS>
struct Ring {
    static constexpr int W = HD * BITS / 8, CH = W / 16, NB = HD / kBlock;
    static constexpr int PITCH = CH % 2 ? W : W + 16;
    static constexpr int V = kGroup * PITCH, KS = 2 * V, VS = KS + kGroup * NB, STAGE = VS + kGroup * NB;
    static constexpr int WARP = kStages * STAGE;
    static constexpr int STATES = kWarps * kQ * (HD + 2) * 4;           // the warps' states, over the rings
    static constexpr int BYTES = (kWarps * WARP > STATES ? kWarps * WARP : STATES);
};

template <int HD, int BITS>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(Cache c, AttnArgs a) {
    using R = Ring<HD, BITS>;
    constexpr int NB = R::NB;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int live[kWarps][kStages];                   // keys of a group that count
    const int split = blockIdx.x, chunks = (a.group + kQ - 1) / kQ;
    const int kh = blockIdx.y / chunks, q0 = (blockIdx.y % chunks) * kQ, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int nq = min(kQ, a.group - q0);
    const int64_t len = length_of(a, c.page_size, b);
    constexpr int kStep = kWarps * kGroup;
    const int64_t per = ((len + a.splits - 1) / a.splits + kStep - 1) / kStep * kStep;
    const int64_t k0 = min(len, split * per), k1 = min(len, k0 + per);

    // query g of this lane as the B fragments of S: per block four f16 pairs of channels t * 8 ...
    uint32_t q[NB][4];
    float c0, c1;                                           // score units of queries 2t and 2t + 1
    {
        float f[NB][8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
            if (g < nq) load8(a.q + b * a.ldq + (int64_t)(kh * a.group + q0 + g) * HD + i * 32 + t * 8, f[i]);
            top = max(top, amax8(f[i]));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = top >> 23;
        const uint32_t up = e == 0 || e == 255 ? 127u : min(253u, 267u - e);    // exponent field of the factor
        const float unit = __uint_as_float((254u - up) << 23) * a.scale_log2;
        c0 = __shfl_sync(0xffffffffu, unit, 8 * t);
        c1 = __shfl_sync(0xffffffffu, unit, 8 * t + 4);
        const float fac = __uint_as_float(up << 23);
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) q[i][j] = pack_f16(f[i][2 * j] * fac, f[i][2 * j + 1] * fac);
    }

    uint8_t* ring = smem + warp * R::WARP;
    const int n = (int)((k1 - k0 + kGroup - 1) / kGroup);   // groups of the split
    const int mine = n > warp ? (n - warp + kWarps - 1) / kWarps : 0;
    const int32_t* table = a.table + b * a.ldt;
    int pages = -1;                                         // lane i: page of this warp's group 32j + i
    auto issue = [&](int i) {                               // copy group i of this warp, if there is one
        if (i < mine) {
            if ((i & 31) == 0) {
                const int64_t key = k0 + (int64_t)(warp + kWarps * (i + lane)) * kGroup;
                pages = key < k1 ? __ldg(table + (key >> c.page_shift)) : -1;
            }
            const int page = __shfl_sync(0xffffffffu, pages, i & 31);
            const int64_t key = k0 + (int64_t)(warp + kWarps * i) * kGroup;
            const bool there = page >= 0 && page < c.pages;
            const int s = i % kStages;
            if (lane == 0) {
                live[warp][s] = there ? (int)min((int64_t)kGroup, k1 - key) : 0;
                if (!there) atomicExch(&g_kvcache_error, kErrIndex);
            }
            if (there) {
                const int64_t row = ((int64_t)page * c.heads + kh) * c.page_size + (key & (c.page_size - 1));
                const uint32_t dst = tc::smem_u32(ring + s * R::STAGE);
                const uint8_t *ks = c.k + row * R::W, *vs = c.v + row * R::W;
#pragma unroll
                for (int j = 0; j < (kGroup * R::CH + 31) / 32; ++j) {
                    const int chunk = lane + 32 * j;
                    if (kGroup * R::CH % 32 == 0 || chunk < kGroup * R::CH) {
                        const uint32_t to = dst + chunk / R::CH * R::PITCH + chunk % R::CH * 16;
                        cp_async16(to, ks + chunk * 16);
                        cp_async16(to + R::V, vs + chunk * 16);
                    }
                }
                const int part = lane & 15;
                if (part < NB)
                    cp_async16(dst + (lane < 16 ? R::KS : R::VS) + part * 16,
                               (lane < 16 ? c.ks : c.vs) + row * NB + part * 16);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;   // of queries 2t and 2t + 1
    float o[2 * NB][4];
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);
    for (int i = 0; i < mine; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        issue(i + kStages - 1);                             // into the stage the last step has read
        uint8_t* st = ring + (i % kStages) * R::STAGE;
        const int nl = live[warp][i % kStages];
        if (nl == 0) continue;
        if (nl < kGroup) {
            // keys past the end: their values and scales, whatever they hold, must not reach the sums
            for (int r = nl; r < kGroup; ++r) {
                for (int j = lane; j < R::W / 4; j += 32) *reinterpret_cast<uint32_t*>(st + R::V + r * R::PITCH + j * 4) = 0;
                if (lane < NB) st[R::VS + r * NB + lane] = 0;
            }
            __syncwarp();
        }
        // S = K Q^T: this lane has keys g and g + 8 of queries 2t and 2t + 1
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            uint32_t ka[4], kb[4];
            const uint8_t* p = st + g * R::PITCH + (k * 32 + t * 8) * BITS / 8;
            key_pairs<BITS>(p, ka);
            key_pairs<BITS>(p + 8 * R::PITCH, kb);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t f0[4] = {ka[0], kb[0], ka[1], kb[1]}, f1[4] = {ka[2], kb[2], ka[3], kb[3]};
            mma_f16(d, f0, q[k][0], q[k][1]);
            mma_f16(d, f1, q[k][2], q[k][3]);
            const float sa = scale_value(st[R::KS + g * NB + k]), sb = scale_value(st[R::KS + (g + 8) * NB + k]);
            s[0] = fmaf(d[0], sa, s[0]);
            s[1] = fmaf(d[1], sa, s[1]);
            s[2] = fmaf(d[2], sb, s[2]);
            s[3] = fmaf(d[3], sb, s[3]);
        }
        s[0] = g < nl ? s[0] * c0 : -INFINITY;
        s[1] = g < nl ? s[1] * c1 : -INFINITY;
        s[2] = g + 8 < nl ? s[2] * c0 : -INFINITY;
        s[3] = g + 8 < nl ? s[3] * c1 : -INFINITY;
        const float t0 = fmaxf(s[0], s[2]), t1 = fmaxf(s[1], s[3]);
        if (__any_sync(0xffffffffu, t0 > m0 + 1.f || t1 > m1 + 1.f)) {
            float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
                n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, w));
                n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, w));
            }
            const float f0 = n0 == -INFINITY ? 1.f : exp2f(m0 - n0), f1 = n1 == -INFINITY ? 1.f : exp2f(m1 - n1);
            m0 = n0;
            m1 = n1;
            l0 *= f0;
            l1 *= f1;
#pragma unroll
            for (int j = 0; j < 2 * NB; ++j) {
                o[j][0] *= f0;
                o[j][1] *= f1;
                o[j][2] *= f0;
                o[j][3] *= f1;
            }
        }
        const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
        const float p[4] = {exp2f(s[0] - r0), exp2f(s[1] - r1), exp2f(s[2] - r0), exp2f(s[3] - r1)};
        l0 += p[0] + p[2];
        l1 += p[1] + p[3];
        // O += V^T P
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const uint32_t ea = st[R::VS + g * NB + k], eb = st[R::VS + (g + 8) * NB + k];
            uint32_t top = max(ea, eb);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, w));
            // 2^14 * 2^(e - top), 0 below the smallest normal number
            const float fa = __uint_as_float((uint32_t)max(141 + (int)ea - (int)top, 0) << 23);
            const float fb = __uint_as_float((uint32_t)max(141 + (int)eb - (int)top, 0) << 23);
            const uint32_t b0 = transpose8(pack_f16(p[0] * fa, p[1] * fa));
            const uint32_t b1 = transpose8(pack_f16(p[2] * fb, p[3] * fb));
            uint32_t va[4], vb[4];                          // keys 2t, 2t + 1 and 2t + 8, 2t + 9
            const uint8_t* v = st + R::V + 2 * t * R::PITCH + (k * 32 + g * 4) * BITS / 8;
            value_pairs<BITS>(v, v + R::PITCH, va);
            value_pairs<BITS>(v + 8 * R::PITCH, v + 9 * R::PITCH, vb);
            const float unit = scale_value(top) * 6.103515625e-05f;             // 2^-14
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t f[4] = {va[2 * h], va[2 * h + 1], vb[2 * h], vb[2 * h + 1]};
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16(d, f, b0, b1);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[2 * k + h][j] = fmaf(d[j], unit, o[2 * k + h][j]);
            }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // join the warps through shared memory
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, w);
        l1 += __shfl_xor_sync(0xffffffffu, l1, w);
    }
    __syncthreads();                                        // the rings are done with
    float* ml = reinterpret_cast<float*>(smem);             // [warp][query][2]
    float* so = ml + kWarps * kQ * 2;                       // [warp][query][HD]
    if (g == 0) {
        float* x = ml + (warp * kQ + 2 * t) * 2;
        x[0] = m0;
        x[1] = l0;
        x[2] = m1;
        x[3] = l1;
    }
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j) {
        float* x = so + (warp * kQ + 2 * t) * HD + j / 2 * 32 + g * 4 + (j & 1) * 2;
        *reinterpret_cast<float2*>(x) = make_float2(o[j][0], o[j][2]);
        *reinterpret_cast<float2*>(x + HD) = make_float2(o[j][1], o[j][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nq * HD; i += kWarps * 32) {
        const int j = i / HD, e = i - j * HD;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ml[(w * kQ + j) * 2]);
        float acc = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float mw = ml[(w * kQ + j) * 2];
            const float f = mw == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : exp2f(mw - mm);
            acc += so[(w * kQ + j) * HD + e] * f;
            ll += ml[(w * kQ + j) * 2 + 1] * f;
        }
        const int h = kh * a.group + q0 + j;
        if (a.splits == 1) {
            a.out[b * a.ldo + (int64_t)h * HD + e] = f2bf(ll == 0.f ? 0.f : acc / ll);
        } else {
            float* x = a.ws + (((int64_t)b * a.heads + h) * a.splits + split) * (2 + HD);
            x[2 + e] = acc;
            if (e == 0) {
                x[0] = mm;
                x[1] = ll;
            }
        }
    }
}

// joins the splits of one (sequence, head); no keys give zeros
template <int HD>
__global__ void __launch_bounds__(HD) combine_kernel(AttnArgs a) {
    __shared__ float weight[kMaxSplits];
    __shared__ float red[2][HD / 32];
    const int h = blockIdx.x, b = blockIdx.y, e = threadIdx.x, warp = e >> 5, lane = e & 31;
    const float* base = a.ws + ((int64_t)b * a.heads + h) * a.splits * (2 + HD);
    float mm = -INFINITY;
    for (int i = e; i < a.splits; i += HD) mm = fmaxf(mm, base[i * (2 + HD)]);
    mm = warp_max(mm);
    if (lane == 0) red[0][warp] = mm;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < HD / 32; ++w) mm = fmaxf(mm, red[0][w]);
    float ll = 0.f;
    for (int i = e; i < a.splits; i += HD) {
        const float mi = base[i * (2 + HD)];
        const float f = mi == -INFINITY ? (mm == -INFINITY ? 1.f : 0.f) : exp2f(mi - mm);
        weight[i] = f;
        ll += base[i * (2 + HD) + 1] * f;
    }
    ll = warp_sum(ll);
    if (lane == 0) red[1][warp] = ll;
    __syncthreads();
    ll = 0.f;
#pragma unroll
    for (int w = 0; w < HD / 32; ++w) ll += red[1][w];
    float acc = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.splits; ++i) acc = fmaf(base[i * (2 + HD) + 2 + e], weight[i], acc);
    a.out[b * a.ldo + (int64_t)h * HD + e] = f2bf(ll == 0.f ? 0.f : acc / ll);
}

// Splits of a sequence's keys: two rounds of the CTAs that fit the GPU (3 of 4 warps on each of 148
// SMs), none with fewer than 128 keys of the longest sequence.
int choose_splits(int batch, int heads, int kv_heads, int64_t longest) {
    const int group = heads / kv_heads;
    const int64_t ctas = (int64_t)batch * kv_heads * ((group + kQ - 1) / kQ);
    const int64_t want = (6 * 148 + ctas - 1) / ctas, by_len = (longest + 127) / 128;
    const int64_t s = want < by_len ? want : by_len;
    return (int)(s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s);
}

constexpr int kMaxDevices = 64;

template <int HD, int BITS>
int launch_attend(const Cache& c, const AttnArgs& a, int batch, cudaStream_t s) {
    static std::atomic<bool> ready[kMaxDevices];            // the kernel's shared memory size is set, per device
    constexpr int bytes = Ring<HD, BITS>::BYTES;
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= kMaxDevices)) return VDIT_ERR_UNSUPPORTED;
    if (e == cudaSuccess && bytes > 48 * 1024 && !ready[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(attend_kernel<HD, BITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) ready[dev].store(true, std::memory_order_release);
    }
    if (e != cudaSuccess) {
        record_cuda_error(e);
        return VDIT_ERR_LAUNCH;
    }
    const dim3 grid(a.splits, c.heads * ((a.group + kQ - 1) / kQ), batch);
    attend_kernel<HD, BITS><<<grid, kWarps * 32, bytes, s>>>(c, a);
    count_launches(1);
    if (a.splits > 1) {
        combine_kernel<HD><<<dim3(a.heads, batch), HD, 0, s>>>(a);
        count_launches(1);
    }
    return check_launch();
}

// the cache's own checks; fills c
int check_cache(void* k, void* v, void* ks, void* vs, int64_t pages, int32_t page_size, int32_t heads, int32_t hd,
                int32_t bits, Cache* c) {
    if (!k || !v || !ks || !vs || pages < 1 || page_size < 1 || heads < 1 || hd < 1) return VDIT_ERR_ARG;
    if ((bits != 4 && bits != 8) || hd % 32 || hd > 128 || (page_size & (page_size - 1)) || page_size < 16 || page_size > 1024 ||
        heads > 4096 || pages > INT32_MAX)
        return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(k) || !aligned16(v) || !aligned16(ks) || !aligned16(vs)) return VDIT_ERR_ALIGN;
    int shift = 0;
    while ((1 << shift) < page_size) ++shift;
    *c = Cache{static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), static_cast<uint8_t*>(ks), static_cast<uint8_t*>(vs),
               pages, page_size, shift, heads, hd};
    return VDIT_OK;
}

// blocks of a launch over n rows of the cache's width, or 0 when they do not fit a grid
int64_t row_blocks(const Cache& c, int64_t n) {
    const int64_t per_row = (int64_t)c.heads * c.hd / 8;
    const int64_t blocks = n > INT64_MAX / per_row - kThreads ? 0 : (n * per_row + kThreads - 1) / kThreads;
    return blocks <= (int64_t)INT32_MAX ? blocks : 0;
}

}  // namespace
}  // namespace kv

int kvcache_error_word(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_kvcache_error, sizeof(int)) != cudaSuccess) return VDIT_ERR_LAUNCH;
    if (clear) {
        int z = 0;
        if (cudaMemcpyToSymbol(g_kvcache_error, &z, sizeof(int)) != cudaSuccess) return VDIT_ERR_LAUNCH;
    }
    return v;
}

}  // namespace vdit

using namespace vdit;
using namespace vdit::kv;

extern "C" int vdit_kv_cache_write(const void* k, int64_t ldk, const void* v, int64_t ldv, const int64_t* slots,
                                   int64_t n, void* kc, void* vc, void* k_scales, void* v_scales, int64_t pages,
                                   int32_t page_size, int32_t heads, int32_t head_dim, int32_t bits,
                                   vdit_stream_t stream) {
    Cache c;
    const int rc = check_cache(kc, vc, k_scales, v_scales, pages, page_size, heads, head_dim, bits, &c);
    if (rc != VDIT_OK) return rc;
    if (!k || !v || !slots || n < 0 || ldk < heads * head_dim || ldv < heads * head_dim) return VDIT_ERR_ARG;
    if (!aligned16(k) || !aligned16(v) || ldk % 8 || ldv % 8) return VDIT_ERR_ALIGN;
    if (n == 0) return VDIT_OK;
    const int64_t blocks = row_blocks(c, n);
    if (!blocks) return VDIT_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const auto* kp = static_cast<const __nv_bfloat16*>(k);
    const auto* vp = static_cast<const __nv_bfloat16*>(v);
    if (bits == 4) write_kernel<4><<<(unsigned)blocks, kThreads, 0, s>>>(kp, ldk, vp, ldv, slots, n, c);
    else write_kernel<8><<<(unsigned)blocks, kThreads, 0, s>>>(kp, ldk, vp, ldv, slots, n, c);
    count_launches(1);
    return check_launch();
}

extern "C" int vdit_kv_cache_read(const void* kc, const void* vc, const void* k_scales, const void* v_scales,
                                  int64_t pages, int32_t page_size, int32_t heads, int32_t head_dim, int32_t bits,
                                  const int64_t* slots, int64_t n, void* k, int64_t ldk, void* v, int64_t ldv,
                                  int32_t out_type, vdit_stream_t stream) {
    Cache c;
    const int rc = check_cache(const_cast<void*>(kc), const_cast<void*>(vc), const_cast<void*>(k_scales),
                               const_cast<void*>(v_scales), pages, page_size, heads, head_dim, bits, &c);
    if (rc != VDIT_OK) return rc;
    if (!k || !v || !slots || n < 0 || ldk < heads * head_dim || ldv < heads * head_dim) return VDIT_ERR_ARG;
    if (out_type != VDIT_BF16 && out_type != VDIT_F32) return VDIT_ERR_ARG;
    const int per16 = out_type == VDIT_F32 ? 4 : 8;
    if (!aligned16(k) || !aligned16(v) || ldk % per16 || ldv % per16) return VDIT_ERR_ALIGN;
    if (n == 0) return VDIT_OK;
    const int64_t blocks = row_blocks(c, n);
    if (!blocks) return VDIT_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto run = [&](auto* kp, auto* vp) {
        if (bits == 4) read_kernel<4><<<(unsigned)blocks, kThreads, 0, s>>>(c, slots, n, kp, ldk, vp, ldv);
        else read_kernel<8><<<(unsigned)blocks, kThreads, 0, s>>>(c, slots, n, kp, ldk, vp, ldv);
    };
    if (out_type == VDIT_F32) run(static_cast<float*>(k), static_cast<float*>(v));
    else run(static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v));
    count_launches(1);
    return check_launch();
}

extern "C" size_t vdit_attention_1q_cached_workspace_bytes(int32_t batch, int32_t heads, int32_t kv_heads,
                                                           int32_t head_dim, int32_t max_pages, int32_t page_size) {
    if (batch < 1 || kv_heads < 1 || heads < kv_heads || head_dim < 1 || max_pages < 1 || page_size < 1) return 0;
    const int splits = choose_splits(batch, heads, kv_heads, (int64_t)max_pages * page_size);
    return splits == 1 ? 0 : (size_t)batch * heads * splits * (2 + head_dim) * sizeof(float);
}

extern "C" int vdit_attention_1q_cached(const void* q, int64_t ldq, const void* kc, const void* vc,
                                        const void* k_scales, const void* v_scales, int64_t pages, int32_t page_size,
                                        int32_t kv_heads, int32_t head_dim, int32_t bits, const int32_t* page_table,
                                        int64_t ld_table, int32_t max_pages, const int32_t* lengths, int32_t batch,
                                        int32_t heads, float softmax_scale, void* out, int64_t ldo, void* workspace,
                                        size_t workspace_bytes, vdit_stream_t stream) {
    Cache c;
    const int rc = check_cache(const_cast<void*>(kc), const_cast<void*>(vc), const_cast<void*>(k_scales),
                               const_cast<void*>(v_scales), pages, page_size, kv_heads, head_dim, bits, &c);
    if (rc != VDIT_OK) return rc;
    if (!q || !page_table || !lengths || !out || batch < 0 || heads < 1 || heads % kv_heads || max_pages < 1 ||
        ld_table < 0 || ldq < (int64_t)heads * head_dim || ldo < (int64_t)heads * head_dim)
        return VDIT_ERR_ARG;
    if (batch > 65535 || heads > 65535) return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(q) || ldq % 8) return VDIT_ERR_ALIGN;
    if (batch == 0) return VDIT_OK;
    const int splits = choose_splits(batch, heads, kv_heads, (int64_t)max_pages * page_size);
    if (workspace_bytes < vdit_attention_1q_cached_workspace_bytes(batch, heads, kv_heads, head_dim, max_pages, page_size) ||
        (splits > 1 && !workspace))
        return VDIT_ERR_WORKSPACE;
    const AttnArgs a{static_cast<const __nv_bfloat16*>(q), ldq, static_cast<__nv_bfloat16*>(out), ldo, page_table,
                     ld_table, lengths, max_pages, heads, heads / kv_heads, splits,
                     softmax_scale * 1.4426950408889634f, static_cast<float*>(workspace)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto run = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        return bits == 4 ? launch_attend<HD, 4>(c, a, batch, s) : launch_attend<HD, 8>(c, a, batch, s);
    };
    if (head_dim == 32) return run(std::integral_constant<int, 32>{});
    if (head_dim == 64) return run(std::integral_constant<int, 64>{});
    if (head_dim == 96) return run(std::integral_constant<int, 96>{});
    return run(std::integral_constant<int, 128>{});
}
