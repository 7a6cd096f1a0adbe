// A paged key/value cache in microscaled 8- or 4-bit floating point (mx.cuh): written as rows
// arrive, read back as rows, and attended to by one query per sequence and head.
//
// Layout: slot = page * page_size + offset.  Keys (and, apart, values) are
// [pages, heads, page_size, head_dim * bits / 8] bytes and their scales
// [pages, heads, page_size, head_dim / 32] bytes, so the keys of one head in one page are
// consecutive: what one query head reads.
#include <math.h>

#include "mx.cuh"
#include "tc.cuh"

namespace vdit {

__device__ int g_kvcache_error = 0;

namespace kv {
namespace {

using namespace mx;

constexpr int kErrIndex = 0x4B56;   // "KV": a slot, page or length outside the cache
constexpr int kThreads = 256;

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
// head_dim * bits / 8 + head_dim / 32 bytes a key, twice, bound by HBM.  A CTA takes one
// sequence, one key head, up to GT of the queries that share it and one range ("split") of the
// sequence's keys.  A lane holds 16 channels (one load of 16 or 8 bytes; half a block, so one
// scale), LPK lanes a key, and every group of LPK lanes runs its own online softmax in fp32 over
// the keys it sees; the groups' states (max, sum, weighted values) are joined once at the end.
constexpr int kWarps = 4;
constexpr int kUnroll = 4;                   // keys in flight per lane: 2 x kUnroll loads

template <int HD> constexpr int lanes_per_key() { return HD == 32 ? 2 : HD == 64 ? 4 : 8; }

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

// 16 channels' codes -> 8 f16 pairs
template <int BITS> struct Codes;
template <> struct Codes<8> {
    uint4 u;
    __device__ __forceinline__ void load(const uint8_t* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
    __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void decode(__half2* h) const {
        decode4_e4m3(u.x, h);
        decode4_e4m3(u.y, h + 2);
        decode4_e4m3(u.z, h + 4);
        decode4_e4m3(u.w, h + 6);
    }
};
template <> struct Codes<4> {
    uint2 u;
    __device__ __forceinline__ void load(const uint8_t* p) { u = __ldg(reinterpret_cast<const uint2*>(p)); }
    __device__ __forceinline__ void zero() { u = make_uint2(0, 0); }
    __device__ __forceinline__ void decode(__half2* h) const {
        decode8_e2m1(u.x, h);
        decode8_e2m1(u.y, h + 4);
    }
};

template <int HD, int BITS, int GT>
__global__ void __launch_bounds__(kWarps * 32) attend_kernel(Cache c, AttnArgs a) {
    constexpr int LPK = lanes_per_key<HD>(), KPW = 32 / LPK, KEYS = kWarps * KPW;
    const int split = blockIdx.x, chunks = (a.group + GT - 1) / GT;
    const int kh = blockIdx.y / chunks, g0 = (blockIdx.y % chunks) * GT, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, li = lane % LPK;
    const bool active = li * 16 < HD;
    const int ng = min(GT, a.group - g0);                   // live queries of this CTA
    const int64_t len = length_of(a, c.page_size, b);
    const int64_t per = ((len + a.splits - 1) / a.splits + KEYS - 1) / KEYS * KEYS;
    const int64_t k0 = min(len, split * per), k1 = min(len, k0 + per);

    float2 q[GT][8];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = 0.f;
        if (active && g < ng) {
            const __nv_bfloat16* p = a.q + b * a.ldq + (int64_t)(kh * a.group + g0 + g) * HD + li * 16;
            load8(p, f);
            load8(p + 8, f + 8);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) q[g][j] = make_float2(f[2 * j] * a.scale_log2, f[2 * j + 1] * a.scale_log2);
    }
    float m[GT], l[GT];
    float2 o[GT][8];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[g][j] = make_float2(0.f, 0.f);
    }

    const int32_t* table = a.table + b * a.ldt;
    // the loop bound is uniform across the warp (the shuffles below need every lane)
    for (int64_t wbase = k0 + warp * KPW; wbase < k1; wbase += (int64_t)KEYS * kUnroll) {
        Codes<BITS> kc[kUnroll], vc[kUnroll];
        uint32_t ksb[kUnroll], vsb[kUnroll];
        bool ok[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int64_t key = wbase + lane / LPK + u * KEYS;
            ok[u] = key < k1;
            int page = -1;
            if (ok[u]) {
                page = __ldg(table + (key >> c.page_shift));
                if (page < 0 || page >= c.pages) {          // no such page: its keys are left out
                    atomicExch(&g_kvcache_error, kErrIndex);
                    ok[u] = false;
                }
            }
            kc[u].zero();
            vc[u].zero();
            ksb[u] = vsb[u] = 0;
            if (ok[u] && active) {
                const int off = (int)(key & (c.page_size - 1));
                const int64_t d = data_at<BITS>(c, page, kh, off) + li * 16 * BITS / 8;
                const int64_t s = scale_at(c, page, kh, off) + li / 2;
                kc[u].load(c.k + d);
                vc[u].load(c.v + d);
                ksb[u] = __ldg(c.ks + s);
                vsb[u] = __ldg(c.vs + s);
            }
        }
        float s[kUnroll][GT];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            __half2 h[8];
            kc[u].decode(h);
            const float sc = scale_value(ksb[u]);
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                for (int j = 0; j < 8; ++j) acc = tc::ffma2v(q[g][j], __half22float2(h[j]), acc);
                float t = (acc.x + acc.y) * sc;
#pragma unroll
                for (int w = LPK / 2; w > 0; w >>= 1) t += __shfl_xor_sync(0xffffffffu, t, w);
                s[u][g] = ok[u] ? t : -INFINITY;
            }
        }
        float p[kUnroll][GT];
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            float mn = m[g];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) mn = fmaxf(mn, s[u][g]);
            const float ref = mn == -INFINITY ? 0.f : mn;   // nothing seen yet: every weight is 0
            const float f = exp2f(m[g] - ref);
            l[g] *= f;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[g][j] = make_float2(o[g][j].x * f, o[g][j].y * f);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                p[u][g] = exp2f(s[u][g] - ref);
                l[g] += p[u][g];
            }
            m[g] = mn;
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            __half2 h[8];
            vc[u].decode(h);
            const float sc = scale_value(vsb[u]);
#pragma unroll
            for (int g = 0; g < GT; ++g) {
                const float w = p[u][g] * sc;
#pragma unroll
                for (int j = 0; j < 8; ++j) o[g][j] = tc::ffma2v(__half22float2(h[j]), make_float2(w, w), o[g][j]);
            }
        }
    }

    // join the KPW groups of a warp in registers, then the warps through shared memory
    __shared__ float sm[kWarps][GT], sl[kWarps][GT], so[kWarps][GT][HD];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        float mm = m[g];
#pragma unroll
        for (int w = LPK; w < 32; w <<= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, w));
        const float f = m[g] == -INFINITY ? 0.f : exp2f(m[g] - mm);
        float ll = l[g] * f;
#pragma unroll
        for (int w = LPK; w < 32; w <<= 1) ll += __shfl_xor_sync(0xffffffffu, ll, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float2 t = make_float2(o[g][j].x * f, o[g][j].y * f);
#pragma unroll
            for (int w = LPK; w < 32; w <<= 1) {
                t.x += __shfl_xor_sync(0xffffffffu, t.x, w);
                t.y += __shfl_xor_sync(0xffffffffu, t.y, w);
            }
            if (lane < LPK && active) {
                so[warp][g][li * 16 + 2 * j] = t.x;
                so[warp][g][li * 16 + 2 * j + 1] = t.y;
            }
        }
        if (lane == 0) {
            sm[warp][g] = mm;
            sl[warp][g] = ll;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ng * HD; i += kWarps * 32) {
        const int g = i / HD, e = i - g * HD;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm[w][g]);
        float acc = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = sm[w][g] == -INFINITY ? 0.f : exp2f(sm[w][g] - mm);
            acc += so[w][g][e] * f;
            ll += sl[w][g] * f;
        }
        const int h = kh * a.group + g0 + g;
        if (a.splits == 1) {
            a.out[b * a.ldo + (int64_t)h * HD + e] = f2bf(len == 0 ? 0.f : acc / ll);
        } else {
            float* p = a.ws + (((int64_t)b * a.heads + h) * a.splits + split) * (2 + HD);
            p[2 + e] = acc;
            if (e == 0) {
                p[0] = mm;
                p[1] = ll;
            }
        }
    }
}

// joins the splits of one (sequence, head); a sequence without keys gives zeros
template <int HD>
__global__ void __launch_bounds__(HD) combine_kernel(AttnArgs a, int page_size) {
    const int h = blockIdx.x, b = blockIdx.y, e = threadIdx.x;
    const float* base = a.ws + ((int64_t)b * a.heads + h) * a.splits * (2 + HD);
    float mm = -INFINITY;
    for (int i = 0; i < a.splits; ++i) mm = fmaxf(mm, base[i * (2 + HD)]);
    float acc = 0.f, ll = 0.f;
    for (int i = 0; i < a.splits; ++i) {
        const float* p = base + i * (2 + HD);
        const float f = p[0] == -INFINITY ? 0.f : exp2f(p[0] - mm);
        ll += p[1] * f;
        acc += p[2 + e] * f;
    }
    const int64_t len = length_of(a, page_size, b);
    a.out[b * a.ldo + (int64_t)h * HD + e] = f2bf(len == 0 ? 0.f : acc / ll);
}

// queries of a CTA: the group, up to 4 (more would not fit the registers: 32 a query)
int queries_per_cta(int group) { return group >= 3 ? 4 : group; }

// Splits of a sequence's keys: enough CTAs for the whole GPU (8 of 4 warps on each of 148 SMs),
// none with fewer than 128 keys of the longest sequence.
int choose_splits(int batch, int heads, int kv_heads, int64_t longest) {
    const int group = heads / kv_heads, gt = queries_per_cta(group);
    const int64_t ctas = (int64_t)batch * kv_heads * ((group + gt - 1) / gt);
    const int64_t want = (8 * 148 + ctas - 1) / ctas, by_len = (longest + 127) / 128;
    const int64_t s = want < by_len ? want : by_len;
    return (int)(s < 1 ? 1 : s > 1024 ? 1024 : s);
}

template <int HD, int BITS>
void launch_attend(const Cache& c, const AttnArgs& a, int batch, cudaStream_t s) {
    const int gt = queries_per_cta(a.group);
    const dim3 grid(a.splits, c.heads * ((a.group + gt - 1) / gt), batch);
    if (gt == 1) attend_kernel<HD, BITS, 1><<<grid, kWarps * 32, 0, s>>>(c, a);
    else if (gt == 2) attend_kernel<HD, BITS, 2><<<grid, kWarps * 32, 0, s>>>(c, a);
    else attend_kernel<HD, BITS, 4><<<grid, kWarps * 32, 0, s>>>(c, a);
    count_launches(1);
    if (a.splits > 1) {
        combine_kernel<HD><<<dim3(a.heads, batch), HD, 0, s>>>(a, c.page_size);
        count_launches(1);
    }
}

// the cache's own checks; fills c
int check_cache(void* k, void* v, void* ks, void* vs, int64_t pages, int32_t page_size, int32_t heads, int32_t hd,
                int32_t bits, Cache* c) {
    if (!k || !v || !ks || !vs || pages < 1 || page_size < 1 || heads < 1 || hd < 1) return VDIT_ERR_ARG;
    if ((bits != 4 && bits != 8) || hd % 32 || hd > 128 || (page_size & (page_size - 1)) || page_size > 1024 ||
        heads > 4096 || pages > INT32_MAX)
        return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(k) || !aligned16(v)) return VDIT_ERR_ALIGN;
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
        if (bits == 4) launch_attend<HD, 4>(c, a, batch, s);
        else launch_attend<HD, 8>(c, a, batch, s);
    };
    if (head_dim == 32) run(std::integral_constant<int, 32>{});
    else if (head_dim == 64) run(std::integral_constant<int, 64>{});
    else if (head_dim == 96) run(std::integral_constant<int, 96>{});
    else run(std::integral_constant<int, 128>{});
    return check_launch();
}
