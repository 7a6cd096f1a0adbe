// A paged key/value cache in microscaled 8- or 4-bit floating point (mx.cuh): written as rows
// arrive, read back as rows, and attended to by one query per sequence and head.
//
// Layout: slot = page * page_size + offset.  Keys (and, apart, values) are
// [pages, heads, page_size, head_dim * bits / 8] bytes and their scales
// [pages, heads, page_size, head_dim / 32] bytes, so the keys of one head in one page are
// consecutive: what one query head reads, in one copy of 16 keys.  The 16-byte pieces of a key are
// exchanged (swapped_piece) so that this copy lands in shared memory without bank conflicts.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "mx.cuh"
#include "tc.cuh"

namespace vdit {

__device__ int g_kvcache_error = 0;

namespace kv {
namespace {

using namespace mx;

constexpr int kErrIndex = 0x4B56;   // "KV": a slot, page or length outside the cache
constexpr int kErrWait = 0x4B57;    // "KW": a bounded wait for copied keys ran out
constexpr int kThreads = 256;
constexpr int kMaxSplits = 1024;
constexpr int64_t kMaxKeys = INT32_MAX - (1 << 20);          // of one sequence: positions stay int32

struct Cache {
    uint8_t *k, *v, *ks, *vs;
    int64_t pages;
    int page_size, page_shift, heads, hd;
};

// ------------------------------------------------------------------ write and read back
// Streams: a thread takes half a block (16 channels) of the key and the value of kRowsAtOnce rows, all
// its loads before the first store, so a row's channels are read and its codes written by consecutive
// threads.  A CTA takes whole rows (as many as fit 256 threads, times kRowsAtOnce; a wider one in
// steps), so that a thread's place takes no 64-bit division.
constexpr int kRowsAtOnce = 2;
struct Rows {
    int64_t n;
    int per_row, per_cta;                                   // half blocks of a row, rows of a CTA at once
};

// calls body(first row, rows apart, first channel) for the thread's half blocks; rows of n and more are
// the body's to leave out
template <typename F>
__device__ __forceinline__ void each_half(const Rows& r, F&& body) {
    const int mine = threadIdx.x / r.per_row;               // 0 when a row takes all threads
    const int64_t row = (int64_t)blockIdx.x * r.per_cta * kRowsAtOnce + mine;
    if (r.per_row > (int)blockDim.x) {
        for (int i = threadIdx.x; i < r.per_row; i += blockDim.x) body(row, 1, i * 16);
    } else if (mine < r.per_cta && row < r.n) {
        body(row, r.per_cta, ((int)threadIdx.x - mine * r.per_row) * 16);
    }
}

// Which 16-byte piece of a key's row (of CH pieces) holds piece 0: piece p is at p ^ swapped_piece.
// Eight neighbouring rows then have the same piece in different 16-byte columns of the 128 bytes
// that shared memory's banks span.
template <int CH>
__host__ __device__ constexpr int swapped_piece(int row) {
    return CH == 8 ? row & 7 : CH == 4 ? row >> 1 & 3 : CH == 6 || CH == 2 ? row >> 2 & 1 : 0;
}

// a thread's place in the cache
template <int HD, int BITS>
__device__ __forceinline__ void place(const Cache& c, int64_t slot, int ch, int64_t* data, int64_t* scale) {
    const int h = ch / HD, e = ch - h * HD;
    const int64_t at = ((slot >> c.page_shift) * c.heads + h) * c.page_size + (slot & (c.page_size - 1));
    constexpr int W = HD * BITS / 8;
    *data = at * W + ((e * BITS / 8) ^ (swapped_piece<W / 16>((int)(slot & 7)) << 4));
    *scale = at * (HD / kBlock) + e / kBlock;
}

template <int BITS>
__device__ __forceinline__ void put_half(const Half<VDIT_BF16>& x, uint8_t* data, uint8_t* scale) {
    const unsigned pair = 3u << (threadIdx.x & 30);
    uint32_t m = x.amax();
    m = max(m, __shfl_xor_sync(pair, m, 1));
    const uint32_t s = scale_byte<BITS>(m);
    if (BITS == 4) *reinterpret_cast<uint2*>(data) = encode_half_e2m1(x, s);
    else *reinterpret_cast<uint4*>(data) = encode_half_e4m3(x, s);
    if (threadIdx.x % 2 == 0) *scale = (uint8_t)s;
}

template <int HD, int BITS>
__global__ void __launch_bounds__(kThreads) write_kernel(const __nv_bfloat16* k, int64_t ldk,
                                                         const __nv_bfloat16* v, int64_t ldv,
                                                         const int64_t* slots, Rows r, Cache c) {
    after_previous();
    each_half(r, [&](int64_t row0, int apart, int ch) {
        int64_t slot[kRowsAtOnce];
        Half<VDIT_BF16> a[kRowsAtOnce], b[kRowsAtOnce];
#pragma unroll
        for (int u = 0; u < kRowsAtOnce; ++u) {
            const int64_t row = row0 + u * apart;
            slot[u] = -1;
            if (row < r.n) {
                slot[u] = load_after(slots + row);
                a[u].load(k + row * ldk + ch);
                b[u].load(v + row * ldv + ch);
            }
        }
#pragma unroll
        for (int u = 0; u < kRowsAtOnce; ++u) {
            if (slot[u] < 0) continue;                      // both threads of a block agree
            if (slot[u] >= c.pages * c.page_size) {
                atomicExch(&g_kvcache_error, kErrIndex);
                continue;
            }
            int64_t d, s;
            place<HD, BITS>(c, slot[u], ch, &d, &s);
            put_half<BITS>(a[u], c.k + d, c.ks + s);
            put_half<BITS>(b[u], c.v + d, c.vs + s);
        }
    });
}

template <int BITS>
struct HalfCodes {
    uint4 u;
    uint32_t s;
    __device__ __forceinline__ void load(const uint8_t* data, const uint8_t* scale) {
        if (BITS == 8) {
            u = load_after(reinterpret_cast<const uint4*>(data));
        } else {
            const uint2 t = load_after(reinterpret_cast<const uint2*>(data));
            u.x = t.x;
            u.y = t.y;
        }
        s = load_after(scale);
    }
    template <typename T>
    __device__ __forceinline__ void store(T* out) const {
        __half2 h[8];
        if (BITS == 8) {
            decode4_e4m3(u.x, h);
            decode4_e4m3(u.y, h + 2);
            decode4_e4m3(u.z, h + 4);
            decode4_e4m3(u.w, h + 6);
        } else {
            decode8_e2m1(u.x, h);
            decode8_e2m1(u.y, h + 4);
        }
        float f[16];
        const float scale = scale_value(s);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 t = fmul2(__half22float2(h[j]), scale);
            f[2 * j] = t.x;
            f[2 * j + 1] = t.y;
        }
        store_half(out, f);
    }
};

template <int HD, int BITS, typename T>
__global__ void __launch_bounds__(kThreads) read_kernel(Cache c, const int64_t* slots, Rows r,
                                                        T* __restrict__ k, int64_t ldk, T* __restrict__ v,
                                                        int64_t ldv) {
    after_previous();
    each_half(r, [&](int64_t row0, int apart, int ch) {
        int64_t slot[kRowsAtOnce];
        HalfCodes<BITS> a[kRowsAtOnce], b[kRowsAtOnce];
#pragma unroll
        for (int u = 0; u < kRowsAtOnce; ++u) slot[u] = row0 + u * apart < r.n ? load_after(slots + row0 + u * apart) : -1;
#pragma unroll
        for (int u = 0; u < kRowsAtOnce; ++u) {
            a[u] = b[u] = HalfCodes<BITS>{make_uint4(0, 0, 0, 0), 0};
            if (slot[u] >= c.pages * c.page_size) {
                atomicExch(&g_kvcache_error, kErrIndex);
            } else if (slot[u] >= 0) {                      // no such row: zeros
                int64_t d, s;
                place<HD, BITS>(c, slot[u], ch, &d, &s);
                a[u].load(c.k + d, c.ks + s);
                b[u].load(c.v + d, c.vs + s);
            }
        }
#pragma unroll
        for (int u = 0; u < kRowsAtOnce; ++u) {
            const int64_t row = row0 + u * apart;
            if (row >= r.n) continue;
            a[u].store(k + row * ldk + ch);
            b[u].store(v + row * ldv + ch);
        }
    });
}

// ------------------------------------------------------------------ single-query attention
// One query per sequence and head over the cached keys of the sequence's pages: a stream of
// head_dim * bits / 8 + head_dim / 32 bytes a key, twice, bound by HBM once the arithmetic keeps up.
// In fp32 on the CUDA cores it did not (an unpack, a conversion and an FMA an element and query: 312 us
// for 16 sequences of up to 32768 keys, 12 x 128 heads, 8 bits; 53 us for 16 of up to 6082 with four
// queries a key head), so both products run on mma.sync m16n8k16: a pair of elements is one
// conversion to f16 (exact for both element types) and up to 8 queries of a key head share it.
//
// A CTA takes one sequence, one key head, up to 8 of its queries and a share ("split") of the keys.
// Its warps are independent until the end: each takes groups of 32 consecutive keys (two halves of
// 16, each in one page), copied by four bulk copies a half into the warp's own ring.  Per group and
// 32-channel block:
//   S = K Q^T   32 keys x 8 queries, times each key's scale in fp32.  Q is f16 after scaling each
//               query by a power of two that puts its largest channel at 2^15: exact but for
//               channels 2^32 below that one.  What undoes it (and the softmax's scale) goes into the
//               key's scale where it makes numbers smaller and behind the sum where it makes them
//               larger, so that no sum overflows that the score itself does not
//   O += V^T P  channels x queries, accumulated by the MMA; P is 2^(s - m) times the key's
//               value scale over a reference, one for each block and query, that keeps the largest
//               of them below 2^15.  The reference falls as m rises and rises when a weight would
//               pass 2^15 (both move O by the same power of two), so that values however large take
//               no precision from the others where their weight is nothing
// 2^(s - m) goes into P as two f16 parts, its first 11 bits and the rest, so that a weight is off by
// 2^-21 of itself, as by the exponential, and not by f16's 2^-11.  Up to 4 queries a key head have
// the second part in the MMA's columns 4 to 7, which would be empty (SLOTS 4: both parts of P for the
// price of one); 5 to 8 queries take a second MMA (SLOTS 8).
// Channels and keys map to fragment indices so that a lane reads consecutive bytes.  m is raised
// only by a score more than 1 above it (a weight stays below 2): exact, as every term uses the same m.
constexpr int kWarps = 4;
constexpr int kQ = 8;                        // columns of the MMAs
constexpr int kGroup = 32;                   // keys of a group

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
    int splits;                              // key ranges of a sequence
    int cluster;                             // CTAs of a cluster: 1, or all splits of a sequence and head
    float scale_log2;
    float* ws;                               // [batch, heads, splits, 2 + hd] when not in a cluster: m, l, mean
};

// a sequence's length, held inside its table row
__device__ __forceinline__ int64_t length_of(const AttnArgs& a, int page_size, int64_t n) {
    const int64_t most = (int64_t)a.max_pages * page_size;
    if (n < 0 || n > most) {
        atomicExch(&g_kvcache_error, kErrIndex);
        return n < 0 ? 0 : most;
    }
    return n;
}

// the output from the largest score, the sum of the weights and the weighted mean: zeros where there were no
// keys, and not a number where there were and none had any weight (all scores -inf)
__device__ __forceinline__ float joined_output(float m, float l, float mean) {
    return m == -INFINITY ? 0.f : l == 0.f ? __uint_as_float(0x7fffffffu) : mean;
}

// 1 / a sum of weights, within 2 ulp (the sums stay far below 2^126, where this division ends); 0 for none
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : __fdividef(1.f, l); }

// a float of shared memory at the same place in CTA `rank` of the cluster
__device__ __forceinline__ float load_cluster(uint32_t addr, int rank) {
    float x;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(tc::mapa_shared(addr, rank)));
    return x;
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

// the NB scale bytes of a row in one word (NB = 3: two words' neighbours, the second one read for
// nothing in some rows)
template <int NB>
__device__ __forceinline__ uint32_t scale_word(const uint8_t* s, int row) {
    if (NB == 4) return *reinterpret_cast<const uint32_t*>(s + row * 4);
    if (NB == 2) return *reinterpret_cast<const uint16_t*>(s + row * 2);
    if (NB == 1) return s[row];
    const uint32_t* w = reinterpret_cast<const uint32_t*>(s) + (row * 3 >> 2);
    return __funnelshift_r(w[0], w[1], (row * 3 & 3) * 8);
}
// the bytes of a word as 2^(byte - 127), two a conversion; 255 is a NaN
template <int NB>
__device__ __forceinline__ void word_scales(uint32_t w, float* s) {
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.bf16x2.ue8m0x2 %0, a;\n\t"
        "cvt.rn.bf16x2.ue8m0x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
    s[0] = __uint_as_float(lo << 16);
    if (NB > 1) s[1] = __uint_as_float(lo & 0xffff0000u);
    if (NB > 2) s[2] = __uint_as_float(hi << 16);
    if (NB > 3) s[3] = __uint_as_float(hi & 0xffff0000u);
}

// shared memory of a warp's ring and of the whole CTA
template <int HD, int BITS>
struct Ring {
    static constexpr int W = HD * BITS / 8, CH = W / 16, NB = HD / kBlock;
    static constexpr int V = kGroup * W, KS = 2 * V, VS = KS + kGroup * NB, STAGE = VS + kGroup * NB;
    // groups in the ring: what leaves room for three CTAs an SM, up to 4
    static constexpr int STAGES = 19000 / STAGE > 4 ? 4 : 19000 / STAGE;
    static_assert(STAGES >= 2, "");
    static constexpr int WARP = STAGES * STAGE;
    static constexpr int STATES = kWarps * kQ * (HD + 2) * 4;           // the warps' states, over the rings
    static constexpr int BYTES = (kWarps * WARP > STATES ? kWarps * WARP : STATES) + 16;   // scale_word reads past
};

// SLOTS: queries of a CTA, at most
template <int HD, int BITS, int SLOTS>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(Cache c, AttnArgs a) {
    using R = Ring<HD, BITS>;
    constexpr int NB = R::NB, kStages = R::STAGES;
    constexpr int PARTS = kQ / SLOTS == 2 ? 1 : 2;          // of the weights, in MMAs of their own
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float joined[kQ][2];                         // max and sum of the CTA's queries
    __shared__ int live[kWarps][kStages][2];                // keys that count of the halves of a group
    __shared__ uint64_t full[kWarps][kStages];              // a group's copies have arrived
    __shared__ int abort_flag;
    const int split = blockIdx.x, chunks = (a.group + SLOTS - 1) / SLOTS;
    const int kh = blockIdx.y / chunks, q0 = (blockIdx.y % chunks) * SLOTS, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int nq = min(SLOTS, a.group - q0), mine_q = g & (SLOTS - 1);
    if (threadIdx.x < kWarps * kStages) tc::mbar_init(tc::smem_u32(&full[0][0] + threadIdx.x), 1);
    if (threadIdx.x == 0) abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    constexpr int step = kWarps * kGroup;
    after_previous();
    // the query is loaded before the branch on the length, so that the two latencies pass at once
    const int32_t given = load_after(a.lengths + b);
    uint4 raw[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
        raw[i] = mine_q < nq ? load_after(reinterpret_cast<const uint4*>(
                                   a.q + b * a.ldq + (int64_t)(kh * a.group + q0 + mine_q) * HD + i * 32 + t * 8))
                             : make_uint4(0, 0, 0, 0);
    const int len = (int)length_of(a, c.page_size, given);      // an int32, as the caller's
    const int per = ((len + kGroup - 1) / kGroup + a.splits - 1) / a.splits * kGroup;
    const int first = (int)min((int64_t)len, (int64_t)split * per) + warp * kGroup;   // groups at first + i * step ...
    const int end = (int)min((int64_t)len, (int64_t)(split + 1) * per);               // ... below end
    const int mine = first < end ? (end - first + step - 1) / step : 0;

    // query mine_q of this lane as the B fragments of S: per block four f16 pairs of channels t * 8 ...
    uint32_t q[NB][4];
    float2 before, after;                                   // score units of columns 2t and 2t + 1
    {
        float f[NB][8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[i][2 * j] = __uint_as_float(w[j] << 16);
                f[i][2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
            top = max(top, amax8(f[i]));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = top >> 23;
        const uint32_t up = e == 0 || e == 255 ? 127u : min(253u, 269u - e);    // exponent field of the factor
        const float unit = __uint_as_float((254u - up) << 23) * a.scale_log2;
        const float2 c = make_float2(__shfl_sync(0xffffffffu, unit, 8 * t), __shfl_sync(0xffffffffu, unit, 8 * t + 4));
        before = make_float2(fabsf(c.x) <= 1.f ? c.x : 1.f, fabsf(c.y) <= 1.f ? c.y : 1.f);
        after = make_float2(fabsf(c.x) <= 1.f ? 1.f : c.x, fabsf(c.y) <= 1.f ? 1.f : c.y);
        const float fac = __uint_as_float(up << 23);
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) q[i][j] = pack_f16(f[i][2 * j] * fac, f[i][2 * j + 1] * fac);
    }

    uint8_t* ring = smem + warp * R::WARP;
    const int32_t* table = a.table + b * a.ldt;
    int pages = -1;                                         // lane j: page of half j of 16 groups
    // copy group i of this warp, if there is one, to stage s: lanes 0 and 1 a half each
    auto issue = [&](int i, int s) {
        if (i >= mine) return;
        if ((i & 15) == 0) {
            const int j = first + (i + (lane >> 1)) * step + (lane & 1) * 16;
            pages = j < end ? load_after(table + (j >> c.page_shift)) : -1;
        }
        const int h = lane & 1, page = __shfl_sync(0xffffffffu, pages, (i & 15) * 2 + h);
        const int key = first + i * step + h * 16;
        const bool there = key < end && page >= 0 && page < c.pages;
        const uint32_t halves = __popc(__ballot_sync(0xffffffffu, lane < 2 && there));
        const uint32_t bar = tc::smem_u32(&full[warp][s]);
        if (lane == 0) tc::mbar_expect_tx(bar, halves * (16 * 2 * (R::W + NB)));
        if (lane < 2) {
            live[warp][s][h] = there ? min(16, end - key) : 0;
            if (there) {
                const int64_t row = ((int64_t)page * c.heads + kh) * c.page_size + (key & (c.page_size - 1));
                const uint32_t dst = tc::smem_u32(ring + s * R::STAGE);
                tc::bulk_load(dst + h * 16 * R::W, c.k + row * R::W, 16 * R::W, bar);
                tc::bulk_load(dst + R::V + h * 16 * R::W, c.v + row * R::W, 16 * R::W, bar);
                tc::bulk_load(dst + R::KS + h * 16 * NB, c.ks + row * NB, 16 * NB, bar);
                tc::bulk_load(dst + R::VS + h * 16 * NB, c.vs + row * NB, 16 * NB, bar);
            } else if (key < end) {
                atomicExch(&g_kvcache_error, kErrIndex);
            }
        }
    };

    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;   // of columns 2t and 2t + 1
    float o[2 * NB][4];                                     // in units of 1 / inv
    float2 inv[NB];                                         // powers of two, one for each block and query
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
#pragma unroll
    for (int k = 0; k < NB; ++k) inv[k] = make_float2(__uint_as_float(254u << 23), __uint_as_float(254u << 23));
    // O of block k, query c (0: 2t, 1: 2t + 1) in units of another inv, its exponent field moved by `by`
    auto move = [&](int k, int c, float times, int by) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            o[2 * k + e][c] *= times;
            o[2 * k + e][c + 2] *= times;
        }
        float& i = c == 0 ? inv[k].x : inv[k].y;
        i = __uint_as_float(__float_as_uint(i) + ((uint32_t)by << 23));
    };
    const float part_h = t < 2 ? 1.f : -1.f, part_s = t < 2 ? 0.f : 1.f;
    auto field = [&](int k, int c) { return (int)(__float_as_uint(c == 0 ? inv[k].x : inv[k].y) >> 23); };

#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i, i);
    // where in a row this lane's 8 channels of a key and 4 of a value are: within the piece, and the
    // exchange of pieces in its rows (g + 8r; 2t + 8r and the next)
    const int key_at = BITS == 8 ? (t & 1) * 8 : t * 4, value_at = BITS == 8 ? (g & 3) * 4 : g * 2;
    const int key_swap = ((BITS == 8 ? t >> 1 : 0) ^ swapped_piece<R::CH>(g)) << 4;
    const int value_swap[2] = {((BITS == 8 ? g >> 2 : 0) ^ swapped_piece<R::CH>(2 * t)) << 4,
                               ((BITS == 8 ? g >> 2 : 0) ^ swapped_piece<R::CH>(2 * t + 1)) << 4};
    int seen = 0;                                           // whether any key of this warp counted
    int done = 0;                                           // groups worked off
    int cur = 0, next = kStages - 1;                        // the stage of this step and the one its copies go to
    uint32_t phase = 0;                                     // of the stages' barriers
    for (int i = 0; i < mine; ++i, ++done) {
        __syncwarp();                                       // every lane has read the stage that is filled next
        issue(i + kStages - 1, next);
        if (!__all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&full[warp][cur]), phase, &abort_flag, &g_kvcache_error,
                                                   kErrWait)))
            break;
        uint8_t* st = ring + cur * R::STAGE;
        const int nl[2] = {live[warp][cur][0], live[warp][cur][1]};
        next = cur;
        cur = cur == kStages - 1 ? 0 : cur + 1;
        if (cur == 0) phase ^= 1;
        const bool whole = nl[0] + nl[1] == kGroup;
        seen |= nl[0] + nl[1];
        if (!whole) {
            // keys that do not count: their values and scales, whatever is there, must not reach the sums
            for (int r = 0; r < kGroup; ++r) {
                if ((r & 15) < nl[r >> 4]) continue;
                for (int j = lane; j < R::W / 4; j += 32) *reinterpret_cast<uint32_t*>(st + R::V + r * R::W + j * 4) = 0;
                if (lane < NB) st[R::VS + r * NB + lane] = 0;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before a later copy to the stage
            __syncwarp();
        }
        // S = K Q^T: this lane has keys g + 8r of queries 2t and 2t + 1
        float2 s[4];
        float ksc[4][NB], vsc[4][NB];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[r] = make_float2(0.f, 0.f);
            word_scales<NB>(scale_word<NB>(st + R::KS, g + 8 * r), ksc[r]);
            word_scales<NB>(scale_word<NB>(st + R::VS, g + 8 * r), vsc[r]);
        }
#pragma unroll
        for (int k = 0; k < NB; ++k) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t ka[4], kb[4];
                const uint8_t* p = st + (g + 16 * h) * R::W + ((k * 4 * BITS) ^ key_swap) + key_at;
                key_pairs<BITS>(p, ka);
                key_pairs<BITS>(p + 8 * R::W, kb);
                float d[4] = {0.f, 0.f, 0.f, 0.f};
                const uint32_t f0[4] = {ka[0], kb[0], ka[1], kb[1]}, f1[4] = {ka[2], kb[2], ka[3], kb[3]};
                mma_f16(d, f0, q[k][0], q[k][1]);
                mma_f16(d, f1, q[k][2], q[k][3]);
                s[2 * h] = tc::ffma2v(make_float2(d[0], d[1]), fmul2(before, ksc[2 * h][k]), s[2 * h]);
                s[2 * h + 1] = tc::ffma2v(make_float2(d[2], d[3]), fmul2(before, ksc[2 * h + 1][k]), s[2 * h + 1]);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[r] = fmul2(s[r], after);
            if (!whole && g + 8 * (r & 1) >= nl[r >> 1]) s[r] = make_float2(-INFINITY, -INFINITY);
        }
        const float t0 = fmaxf(fmaxf(s[0].x, s[1].x), fmaxf(s[2].x, s[3].x));
        const float t1 = fmaxf(fmaxf(s[0].y, s[1].y), fmaxf(s[2].y, s[3].y));
        if (__any_sync(0xffffffffu, t0 > m0 + 1.f || t1 > m1 + 1.f)) {
            float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
                n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, w));
                n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, w));
            }
            const float f[2] = {n0 == -INFINITY ? 1.f : exp2f(m0 - n0), n1 == -INFINITY ? 1.f : exp2f(m1 - n1)};
            // whole powers of two by which m rises: the references follow (O only shrinks)
            const int rise[2] = {(int)fminf(n0 - m0, 120.f), (int)fminf(n1 - m1, 120.f)};
            m0 = n0;
            m1 = n1;
            l0 *= f[0];
            l1 *= f[1];
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int by = min(254 - field(k, c), rise[c]);
                    move(k, c, f[c] * __uint_as_float((uint32_t)(127 + by) << 23), by);
                }
        }
        const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
        for (int r = 0; r < 4; ++r) {                       // scores to weights
            s[r] = make_float2(tc::ex2(s[r].x - r0), tc::ex2(s[r].y - r1));
            l0 += s[r].x;
            l1 += s[r].y;
        }
        // O += V^T P, one block after another
        auto first = [](float2 y) {                         // 11 bits of each
            return make_float2(__uint_as_float(__float_as_uint(y.x) & 0xffffe000u),
                               __uint_as_float(__float_as_uint(y.y) & 0xffffe000u));
        };
        if (PARTS == 1)                                     // the first part in columns 0 to 3, the rest in 4 to 7
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s[r] = tc::ffma2v(first(s[r]), make_float2(part_h, part_h), fmul2(s[r], part_s));
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            uint32_t pk[PARTS][4];
            auto weights = [&] {                            // as f16 pairs; returns the largest
                uint32_t top = 0;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float2 y = fmul2(fmul2(s[r], vsc[r][k]), inv[k]);
                    const float2 h = PARTS == 1 ? y : first(y);
                    pk[0][r] = pack_f16(h.x, h.y);
                    if (PARTS == 2) {
                        const float2 rest = tc::ffma2v(h, make_float2(-1.f, -1.f), y);
                        pk[PARTS - 1][r] = pack_f16(rest.x, rest.y);
                    }
                    top = __vmaxu2(top, pk[0][r]);          // the first part is the larger one
                }
                return max(top >> 16, top & 0xffffu);
            };
            if (__any_sync(0xffffffffu, weights() > 0x7800u)) {         // 2^15
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float w = 0.f;
#pragma unroll
                    for (int r = 0; r < 4; ++r) w = fmaxf(w, (c == 0 ? s[r].x : s[r].y) * vsc[r][k]);
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, x));
                    // the exponent field that brings w to 2^13 ... 2^14
                    const int by = max(267 - (int)(__float_as_uint(w) >> 23), 1) - field(k, c);
                    if (by < 0) move(k, c, by > -127 ? __uint_as_float((uint32_t)(127 + by) << 23) : 0.f, by);
                }
                weights();
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t b[PARTS][2];
#pragma unroll
                for (int i = 0; i < PARTS; ++i) {
                    b[i][0] = transpose8(pk[i][2 * h]);
                    b[i][1] = transpose8(pk[i][2 * h + 1]);
                }
                uint32_t va[4], vb[4];                      // keys 2t, 2t + 1 and 2t + 8, 2t + 9 of the half
                const uint8_t* v = st + R::V + (2 * t + 16 * h) * R::W + value_at;
                const uint8_t *v0 = v + ((k * 4 * BITS) ^ value_swap[0]), *v1 = v + R::W + ((k * 4 * BITS) ^ value_swap[1]);
                value_pairs<BITS>(v0, v1, va);
                value_pairs<BITS>(v0 + 8 * R::W, v1 + 8 * R::W, vb);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t f[4] = {va[2 * e], va[2 * e + 1], vb[2 * e], vb[2 * e + 1]};
#pragma unroll
                    for (int i = 0; i < PARTS; ++i) mma_f16(o[2 * k + e], f, b[i][0], b[i][1]);
                }
            }
        }
    }
    // after an abort: the copies still on their way land before the ring becomes the place of the states
    if (done < mine)
        tc::drain_loads(done, min(mine, done + kStages), kStages,
                        [&](int s) { return tc::smem_u32(&full[warp][s]); }, &g_kvcache_error, kErrWait);
    // a warp whose scores were all -inf (a query with infinities) has seen keys, unlike an empty one:
    // alone it makes 0 / 0, not zeros
    if (seen) {
        m0 = fmaxf(m0, -FLT_MAX);
        m1 = fmaxf(m1, -FLT_MAX);
    }
    // join the warps through shared memory.  What is joined, here and over the splits, is the largest score m,
    // the sum l of the weights and the weighted mean of the values: sums of values could pass fp32's range
    // where their mean does not
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, w);
        l1 += __shfl_xor_sync(0xffffffffu, l1, w);
    }
    __syncthreads();                                        // the rings are done with
    float* ml = reinterpret_cast<float*>(smem);             // [warp][query][2]
    float* so = ml + kWarps * kQ * 2;                       // [warp][query][HD]
    const bool holds = 2 * t < SLOTS;                       // columns 2t and 2t + 1 are queries
    if (g == 0 && holds) {
        float* x = ml + (warp * kQ + 2 * t) * 2;
        x[0] = m0;
        x[1] = l0;
        x[2] = m1;
        x[3] = l1;
    }
    const float n0 = inverse(l0), n1 = inverse(l1);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
        const float u0 = __uint_as_float(max((uint32_t)(254 - field(k, 0)) << 23, 0x00400000u));      // 1 / inv
        const float u1 = __uint_as_float(max((uint32_t)(254 - field(k, 1)) << 23, 0x00400000u));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float* x = o[2 * k + e];
            float2 v0 = make_float2(x[0] * n0 * u0, x[2] * n0 * u0), v1 = make_float2(x[1] * n1 * u1, x[3] * n1 * u1);
            if (PARTS == 1) {                               // the weights' second parts, of columns 4 to 7
                v0 = tc::fadd2(v0, make_float2(__shfl_down_sync(0xffffffffu, v0.x, 2), __shfl_down_sync(0xffffffffu, v0.y, 2)));
                v1 = tc::fadd2(v1, make_float2(__shfl_down_sync(0xffffffffu, v1.x, 2), __shfl_down_sync(0xffffffffu, v1.y, 2)));
            }
            if (!holds) continue;
            float* to = so + (warp * kQ + 2 * t) * HD + k * 32 + g * 4 + e * 2;
            *reinterpret_cast<float2*>(to) = v0;
            *reinterpret_cast<float2*>(to + HD) = v1;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nq * HD; i += kWarps * 32) {
        const int j = i / HD, e = i - j * HD;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ml[(w * kQ + j) * 2]);
        float acc = 0.f, ll = 0.f, f[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float mw = ml[(w * kQ + j) * 2];
            f[w] = mw == -INFINITY ? 0.f : exp2f(mw - mm) * ml[(w * kQ + j) * 2 + 1];
            ll += f[w];
        }
        const float share = inverse(ll);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) acc = fmaf(so[(w * kQ + j) * HD + e], f[w] * share, acc);
        const int h = kh * a.group + q0 + j;
        if (a.splits == 1) {
            a.out[b * a.ldo + (int64_t)h * HD + e] = f2bf(joined_output(mm, ll, acc));
        } else if (a.cluster == 1) {
            float* x = a.ws + (((int64_t)b * a.heads + h) * a.splits + split) * (2 + HD);
            x[2 + e] = acc;
            if (e == 0) {
                x[0] = mm;
                x[1] = ll;
            }
        } else {
            so[j * HD + e] = acc;                           // in warp 0's place, which no other thread reads
            if (e == 0) {
                joined[j][0] = mm;
                joined[j][1] = ll;
            }
        }
    }
    if (a.cluster == 1) return;
    // the splits of a sequence and head are the CTAs of this cluster: each joins its part of the
    // outputs through distributed shared memory.  A warp's 32 outputs are of one query: lane r has the
    // weight of rank r
    tc::cluster_sync();
    const uint32_t so_at = tc::smem_u32(so), joined_at = tc::smem_u32(joined);
    for (int i = split * kWarps * 32 + threadIdx.x; i < nq * HD; i += a.cluster * kWarps * 32) {
        const int j = i / HD;
        const float mr = lane < a.cluster ? load_cluster(joined_at + j * 8, lane) : -INFINITY;
        const float lr = lane < a.cluster ? load_cluster(joined_at + j * 8 + 4, lane) : 0.f;
        const float mm = warp_max(mr);
        const float f = mr == -INFINITY ? 0.f : exp2f(mr - mm) * lr;
        const float ll = warp_sum(f), share = f * inverse(ll);
        float acc = 0.f;
        for (int r0 = 0; r0 < a.cluster; r0 += 8) {
            float x[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) x[r] = r0 + r < a.cluster ? load_cluster(so_at + i * 4, r0 + r) : 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) acc = fmaf(x[r], __shfl_sync(0xffffffffu, share, r0 + r), acc);
        }
        a.out[b * a.ldo + (int64_t)(kh * a.group + q0) * HD + i] = f2bf(joined_output(mm, ll, acc));
    }
    tc::cluster_sync();                                     // no CTA leaves while another reads its memory
}

// joins the splits of one (sequence, head); no keys give zeros
template <int HD>
__global__ void __launch_bounds__(HD) combine_kernel(AttnArgs a) {
    __shared__ float weight[kMaxSplits];
    __shared__ float red[2][HD / 32];
    const int h = blockIdx.x, b = blockIdx.y, e = threadIdx.x, warp = e >> 5, lane = e & 31;
    const float* base = a.ws + ((int64_t)b * a.heads + h) * a.splits * (2 + HD);
    asm volatile("griddepcontrol.wait;" ::: "memory");      // the splits' states are written
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
        const float f = mi == -INFINITY ? 0.f : exp2f(mi - mm) * base[i * (2 + HD) + 1];
        weight[i] = f;
        ll += f;
    }
    ll = warp_sum(ll);
    if (lane == 0) red[1][warp] = ll;
    __syncthreads();
    ll = 0.f;
#pragma unroll
    for (int w = 0; w < HD / 32; ++w) ll += red[1][w];
    const float share = inverse(ll);
    float acc = 0.f;
#pragma unroll 8
    for (int i = 0; i < a.splits; ++i) acc = fmaf(base[i * (2 + HD) + 2 + e], weight[i] * share, acc);
    a.out[b * a.ldo + (int64_t)h * HD + e] = f2bf(joined_output(mm, ll, acc));
}

// How the keys of a sequence are split: two rounds of 3 CTAs on each of 148 SMs but no fewer than 128 keys
// of the longest sequence, one group a warp; four rounds, for an even end, where a split then still has
// 1024.  3 CTAs are what an SM holds of 128 channels and of 64 in 8 bits; of 96 channels it holds 4, of 64
// in 4 bits 5, of 32 6 or 8, so there a round is a part of one.  Up to 16 splits with no more than 2048 keys
// each, and no more than 4 CTAs an SM in all, are a cluster, which joins them itself (one launch, no
// workspace); otherwise their states go through the workspace to a second kernel (16 sequences of up to
// 32768 keys: 200 us when this was chosen, 191 now; in clusters of 2 or 8 272 and 233 then).
// The longest sequence is the table's width: the lengths are on the GPU.  A table far wider than its
// sequences is planned for as if it were full (16 sequences of up to 300 keys, 12 x 128: 10.4 us in a table of
// 300 or 4096 keys, 21.8 in one of 32768).
// Queries of a CTA, at most: 4 with both parts of their weights in one MMA, 8 with two.  16 sequences over 8
// key heads of 96 channels, 8 bits: 4 queries a key head (up to 20000 keys) 76 us with 4, 81 with 8; 5 queries
// (up to 16000 keys) 105 with 4 (two CTAs read the same keys), 73 with 8.
int slots_of(int group) { return group <= 4 ? 4 : kQ; }

struct Plan {
    int splits, cluster;
};
Plan plan_of(int batch, int heads, int kv_heads, int64_t longest) {
    const int group = heads / kv_heads;
    const int64_t ctas = (int64_t)batch * kv_heads * ((group + slots_of(group) - 1) / slots_of(group));
    const int64_t two = std::min(6 * 148 / ctas, (longest + 127) / 128), four = std::min(12 * 148 / ctas, longest / 1024);
    const int64_t want = std::min<int64_t>(std::max<int64_t>(std::max(two, four), 1), kMaxSplits);
    int c = 1;
    while (c < 16 && c < want && ctas * 2 * c <= 4 * 148) c *= 2;
    if (c >= want || (longest <= (int64_t)c * 2048 && ctas * c >= 148)) return {c, c};
    return {(int)want, 1};
}

constexpr int kMaxDevices = 64;

template <int HD, int BITS, int SLOTS>
int launch_attend(const Cache& c, const AttnArgs& a, int batch, cudaStream_t s) {
    static std::atomic<bool> ready[kMaxDevices];            // the kernel's attributes are set, per device
    constexpr int bytes = Ring<HD, BITS>::BYTES;
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev < 0 || dev >= kMaxDevices)) return VDIT_ERR_UNSUPPORTED;
    if (e == cudaSuccess && !ready[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(attend_kernel<HD, BITS, SLOTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attend_kernel<HD, BITS, SLOTS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) ready[dev].store(true, std::memory_order_release);
    }
    if (e != cudaSuccess) {
        record_cuda_error(e);
        return VDIT_ERR_LAUNCH;
    }
    const dim3 grid(a.splits, c.heads * ((a.group + SLOTS - 1) / SLOTS), batch);
    // Set up while the kernel before it ends.  When this was chosen, 16 ragged sequences took 18.9 us in a stream of
    // calls instead of 20.5 and one of 4101 keys 12.6 either way; replayed in a graph, where launches are
    // close already, the one sequence took 12.4 instead of 11.9 (12.2 now).
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster > 1 ? 2 : 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = bytes;
    e = cudaLaunchKernelEx(&cfg, attend_kernel<HD, BITS, SLOTS>, c, a);
    if (e != cudaSuccess) {
        record_cuda_error(e);
        return VDIT_ERR_LAUNCH;
    }
    count_launches(1);
    if (a.splits > a.cluster) {
        // resident before the splits are done: the launch is hidden behind them
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(a.heads, batch);
        cfg.blockDim = dim3(HD);
        cfg.dynamicSmemBytes = 0;
        e = cudaLaunchKernelEx(&cfg, combine_kernel<HD>, a);
        if (e != cudaSuccess) {
            record_cuda_error(e);
            return VDIT_ERR_LAUNCH;
        }
        count_launches(1);
    }
    return check_launch();
}

// the cache's own checks; fills c
int check_cache(const vdit_kv_cache* v, Cache* c) {
    if (!v || !v->k || !v->v || !v->k_scales || !v->v_scales || v->pages < 1 || v->page_size < 1 || v->heads < 1 ||
        v->head_dim < 1)
        return VDIT_ERR_ARG;
    if ((v->bits != 4 && v->bits != 8) || v->head_dim % 32 || v->head_dim > 128 || (v->page_size & (v->page_size - 1)) ||
        v->page_size < 16 || v->page_size > 1024 || v->heads > 4096 || v->pages > INT32_MAX)
        return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(v->k) || !aligned16(v->v) || !aligned16(v->k_scales) || !aligned16(v->v_scales)) return VDIT_ERR_ALIGN;
    int shift = 0;
    while ((1 << shift) < v->page_size) ++shift;
    *c = Cache{static_cast<uint8_t*>(v->k), static_cast<uint8_t*>(v->v), static_cast<uint8_t*>(v->k_scales),
               static_cast<uint8_t*>(v->v_scales), v->pages, v->page_size, shift, v->heads, v->head_dim};
    return VDIT_OK;
}

// a launch over n rows of the cache's width: CTAs and threads, 0 CTAs when they do not fit a grid
Rows rows_of(const Cache& c, int64_t n, int64_t* ctas, int* threads) {
    const int per_row = c.heads * c.hd / 16, per_cta = per_row < kThreads ? kThreads / per_row : 1;
    *ctas = (n + (int64_t)per_cta * kRowsAtOnce - 1) / (per_cta * kRowsAtOnce);
    if (*ctas > (int64_t)INT32_MAX) *ctas = 0;
    *threads = per_row < kThreads ? (per_row * per_cta + 31) / 32 * 32 : kThreads;
    return {n, per_row, per_cta};
}

// body(head_dim, bits) as constants
template <typename F>
void with_format(int hd, int bits, F&& body) {
    auto sized = [&](auto b) {
        if (hd == 32) body(std::integral_constant<int, 32>{}, b);
        else if (hd == 64) body(std::integral_constant<int, 64>{}, b);
        else if (hd == 96) body(std::integral_constant<int, 96>{}, b);
        else body(std::integral_constant<int, 128>{}, b);
    };
    if (bits == 4) sized(std::integral_constant<int, 4>{});
    else sized(std::integral_constant<int, 8>{});
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
                                   int64_t n, const vdit_kv_cache* cache, vdit_stream_t stream) {
    Cache c;
    const int rc = check_cache(cache, &c);
    if (rc != VDIT_OK) return rc;
    const int d = c.heads * c.hd;
    if (!k || !v || !slots || n < 0 || ldk < d || ldv < d) return VDIT_ERR_ARG;
    if (!aligned16(k) || !aligned16(v) || ldk % 8 || ldv % 8) return VDIT_ERR_ALIGN;
    if (n == 0) return VDIT_OK;
    int64_t ctas;
    int threads;
    const Rows r = rows_of(c, n, &ctas, &threads);
    if (!ctas) return VDIT_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    with_format(c.hd, cache->bits, [&](auto hd, auto bits) {
        launch_early(write_kernel<decltype(hd)::value, decltype(bits)::value>, dim3((unsigned)ctas), threads, s,
                     static_cast<const __nv_bfloat16*>(k), ldk, static_cast<const __nv_bfloat16*>(v), ldv, slots, r, c);
    });
    count_launches(1);
    return check_launch();
}

extern "C" int vdit_kv_cache_read(const vdit_kv_cache* cache, const int64_t* slots, int64_t n, void* k, int64_t ldk,
                                  void* v, int64_t ldv, int32_t out_type, vdit_stream_t stream) {
    Cache c;
    const int rc = check_cache(cache, &c);
    if (rc != VDIT_OK) return rc;
    const int d = c.heads * c.hd;
    if (!k || !v || !slots || n < 0 || ldk < d || ldv < d) return VDIT_ERR_ARG;
    if (out_type != VDIT_BF16 && out_type != VDIT_F32) return VDIT_ERR_ARG;
    const int per16 = out_type == VDIT_F32 ? 4 : 8;
    if (!aligned16(k) || !aligned16(v) || ldk % per16 || ldv % per16) return VDIT_ERR_ALIGN;
    if (n == 0) return VDIT_OK;
    int64_t ctas;
    int threads;
    const Rows r = rows_of(c, n, &ctas, &threads);
    if (!ctas) return VDIT_ERR_UNSUPPORTED;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    with_format(c.hd, cache->bits, [&](auto hd, auto bits) {
        constexpr int HD = decltype(hd)::value, BITS = decltype(bits)::value;
        if (out_type == VDIT_F32)
            launch_early(read_kernel<HD, BITS, float>, dim3((unsigned)ctas), threads, s, c, slots, r,
                         static_cast<float*>(k), ldk, static_cast<float*>(v), ldv);
        else
            launch_early(read_kernel<HD, BITS, __nv_bfloat16>, dim3((unsigned)ctas), threads, s, c, slots, r,
                         static_cast<__nv_bfloat16*>(k), ldk, static_cast<__nv_bfloat16*>(v), ldv);
    });
    count_launches(1);
    return check_launch();
}

extern "C" size_t vdit_attention_1q_cached_workspace_bytes(int32_t batch, int32_t heads, int32_t kv_heads,
                                                           int32_t head_dim, int32_t max_pages, int32_t page_size) {
    if (batch < 1 || kv_heads < 1 || heads < kv_heads || head_dim < 1 || max_pages < 1 || page_size < 1) return 0;
    const int64_t longest = (int64_t)max_pages * page_size;
    if (longest > kMaxKeys) return 0;
    const Plan plan = plan_of(batch, heads, kv_heads, longest);
    return plan.splits == plan.cluster ? 0 : (size_t)batch * heads * plan.splits * (2 + head_dim) * sizeof(float);
}

extern "C" int vdit_attention_1q_cached(const void* q, int64_t ldq, const vdit_kv_cache* cache,
                                        const int32_t* page_table, int64_t ld_table, int32_t max_pages,
                                        const int32_t* lengths, int32_t batch, int32_t heads, float softmax_scale,
                                        void* out, int64_t ldo, void* workspace, size_t workspace_bytes,
                                        vdit_stream_t stream) {
    Cache c;
    const int rc = check_cache(cache, &c);
    if (rc != VDIT_OK) return rc;
    const int kv_heads = c.heads, head_dim = c.hd, page_size = c.page_size;
    if (!q || !page_table || !lengths || !out || batch < 0 || heads < 1 || heads % kv_heads || max_pages < 1 ||
        ld_table < 0 || ldq < (int64_t)heads * head_dim || ldo < (int64_t)heads * head_dim)
        return VDIT_ERR_ARG;
    if (batch > 65535 || heads > 65535 || (int64_t)max_pages * page_size > kMaxKeys)
        return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(q) || ldq % 8) return VDIT_ERR_ALIGN;
    if (batch == 0) return VDIT_OK;
    const int64_t longest = (int64_t)max_pages * page_size;
    const Plan plan = plan_of(batch, heads, kv_heads, longest);
    if (workspace_bytes < vdit_attention_1q_cached_workspace_bytes(batch, heads, kv_heads, head_dim, max_pages, page_size) ||
        (plan.splits > plan.cluster && !workspace))
        return VDIT_ERR_WORKSPACE;
    if (workspace && !aligned16(workspace)) return VDIT_ERR_ALIGN;
    const AttnArgs a{static_cast<const __nv_bfloat16*>(q), ldq, static_cast<__nv_bfloat16*>(out), ldo, page_table,
                     ld_table, lengths, max_pages, heads, heads / kv_heads, plan.splits, plan.cluster,
                     softmax_scale * 1.4426950408889634f, static_cast<float*>(workspace)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int status = VDIT_OK;
    with_format(c.hd, cache->bits, [&](auto hd, auto bits) {
        constexpr int HD = decltype(hd)::value, BITS = decltype(bits)::value;
        status = slots_of(a.group) == 4 ? launch_attend<HD, BITS, 4>(c, a, batch, s) : launch_attend<HD, BITS, kQ>(c, a, batch, s);
    });
    return status;
}
