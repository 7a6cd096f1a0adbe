// PTX wrappers shared by the tcgen05 kernels: mbarriers, TMA, tcgen05 MMA /
// commit / TMEM load-store, packed fp32x2 math and shared-memory matrix
// descriptors (sm_100 format).
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace vdit {
namespace tc {

// ---------------------------------------------------------------- PTX wrappers
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// whether the phase has completed, without waiting (try_wait may suspend the thread for a while)
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// low word of the device's nanosecond timer; it wraps after 4.3 s
__device__ __forceinline__ uint32_t timer_ns() {
    uint32_t t;
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
    return t;
}

// Wait bounded in time.  Returns false when the CTA aborted (another thread's wait ran out) or when
// this wait has lasted kWaitLimitNs; then it raises the CTA abort flag and records `code` in the
// device error word `err`.  A poll suspends the thread for up to 1.3 us (measured; the hardware's own
// limit), so a count of polls would be no bound one can state.  The timer is read after every 256 polls
// of an inner loop with a constant count: 0.306 ms for the depthwise conv of 16384 voxels and 0.408 for
// their attention; with the timer read at each poll 0.317 and 0.413, in one loop with a test 0.316 and 0.410.
constexpr uint32_t kWaitLimitNs = 2000000000u;       // below half the timer word's range
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* err,
                                          int code) {
    uint32_t start = 0;
    for (uint32_t c = 0;; ++c) {
        for (uint32_t i = 0; i < 256; ++i) {
            if (mbar_try_wait(bar, parity)) return true;
            if (*abort_flag) return false;
        }
        const uint32_t now = timer_ns();
        if (c == 0) start = now;
        else if (now - start > kWaitLimitNs) break;
    }
    *abort_flag = 1;
    atomicExch(err, code);
    return false;
}

// The end of an aborted CTA.  Waits (bounded) for the last fills of a ring of loads: fill j went to stage
// j % stages and completes phase j / stages of full(stage).  Called by one thread before the CTA leaves or
// uses the ring for something else, so that no copy lands in memory that is no longer the ring's.
template <typename F>
__device__ __forceinline__ void drain_loads(int first, int issued, int stages, F&& full, int* err, int code) {
    volatile int gave_up = 0;
    for (int j = max(first, issued - stages); j < issued; ++j)
        if (!mbar_wait(full(j % stages), (uint32_t)(j / stages) & 1, &gave_up, err, code)) return;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void tc_mma(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum)
        : "memory");
}

// 32 lanes x 32 consecutive fp32 columns -> 32 registers per thread
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float* v) {
    uint32_t r[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}


// D (TMEM) += A (TMEM) * B (smem descriptor)
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accum)
        : "memory");
}

// Issue from a converged warp: every lane runs the call with the same operands and the lane
// that elect.sync picks (the same one every time for a full mask) issues the MMA or the commit.
// Operands computed by the whole warp stay in uniform registers; the same MMAs issued under
// `if (lane == 0)` with per-tile descriptor arithmetic cost ~80 clocks each (measured), more
// than an M=128, N=128, K=16 MMA takes to execute (64 clocks).
__device__ __forceinline__ void tc_mma_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum)
        : "memory");
}

// as tc_mma_elect with the A operand in tensor memory
__device__ __forceinline__ void tc_mma_ts_elect(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                                uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accum)
        : "memory");
}

// commit by the elected lane: the lane that issued the MMAs of tc_mma_elect / tc_mma_ts_elect
__device__ __forceinline__ void tc_commit_elect(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(bar)
        : "memory");
}

// 32 lanes x 16 consecutive 32-bit columns from 16 registers per thread
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// packed fp32x2 FMA: (a.x*s + b, a.y*s + b)
__device__ __forceinline__ float2 ffma2(float2 a, float s, float b) {
    unsigned long long ra, rs, rb, rd;
    asm("mov.b64 %0, {%1,%2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1,%1};" : "=l"(rs) : "f"(s));
    asm("mov.b64 %0, {%1,%1};" : "=l"(rb) : "f"(b));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(rd) : "l"(ra), "l"(rs), "l"(rb));
    float2 o;
    asm("mov.b64 {%0,%1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(rd));
    return o;
}

__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
    unsigned long long ra, rb, rd;
    asm("mov.b64 %0, {%1,%2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1,%2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
    float2 o;
    asm("mov.b64 {%0,%1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(rd));
    return o;
}

// packed fp32x2 FMA with vector operands: a*b + c
__device__ __forceinline__ float2 ffma2v(float2 a, float2 b, float2 c) {
    unsigned long long ra, rb, rc, rd;
    asm("mov.b64 %0, {%1,%2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
    asm("mov.b64 %0, {%1,%2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
    asm("mov.b64 %0, {%1,%2};" : "=l"(rc) : "f"(c.x), "f"(c.y));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(rd) : "l"(ra), "l"(rb), "l"(rc));
    float2 o;
    asm("mov.b64 {%0,%1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(rd));
    return o;
}

// 2^x on the FMA pipe (for x <= ~16), to take part of the exponentials off
// the MUFU unit.  Range reduction x = j + f with j = round(x) (magic-number
// add), f in [-1/2, 1/2]; 2^f from a degree-3 polynomial fitted here by
// relative-error least squares on Chebyshev nodes (max rel. error 1.2e-4,
// below the bf16 rounding the probabilities get next); 2^j is added to the
// exponent field.  x is clamped at -126 so the exponent never wraps.
__device__ __forceinline__ float2 exp2_fma2(float2 x) {
    constexpr float kMagic = 12582912.0f;          // 1.5 * 2^23
    x.x = fmaxf(x.x, -126.f);
    x.y = fmaxf(x.y, -126.f);
    const float2 t = fadd2(x, make_float2(kMagic, kMagic));
    const float2 j = fadd2(t, make_float2(-kMagic, -kMagic));
    const float2 f = ffma2v(j, make_float2(-1.f, -1.f), x);
    float2 p = ffma2v(f, make_float2(0.05459282547f, 0.05459282547f), make_float2(0.24221783876f, 0.24221783876f));
    p = ffma2v(p, f, make_float2(0.69336861372f, 0.69336861372f));
    p = ffma2v(p, f, make_float2(1.f, 1.f));
    return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// Shared-memory matrix descriptors (sm_100 format: start>>4 in [0,14), LBO>>4 in
// [16,30), SBO>>4 in [32,46), version 1 at bit 46, layout type in [61,64)).
__device__ __forceinline__ uint64_t make_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo, uint64_t layout) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (layout << 61);
}


// Shared-memory matrix descriptor layout types
constexpr uint64_t kSw128 = 2, kSw64 = 4;

// instruction descriptor: f32 accumulate, bf16 A/B, A K-major, B K- or MN-major
__host__ __device__ constexpr uint32_t make_idesc(int m, int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

// ---------------------------------------------------------------- block-scaled 4-bit MMAs
// instruction descriptor of kind::mxf4: f32 accumulate, e2m1 A/B (K-major), ue8m0 scales; sf picks
// the scale bytes (0 or 2: the low or the high two of a TMEM word) of both operands
__host__ __device__ constexpr uint32_t make_idesc_mxf4(int m, int n, int sf) {
    return ((uint32_t)sf << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) |
           ((uint32_t)(m >> 7) << 27) | ((uint32_t)sf << 29);
}

// ---------------------------------------------------------------- CTA pairs (cta_group::2)
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// the shared::cluster address of the same shared-memory object in CTA `cta` of the cluster
__device__ __forceinline__ uint32_t mapa_shared(uint32_t addr, uint32_t cta) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
    return r;
}

// The barrier's aligned form is for whole warps: one of which a single lane has just run a role (a producer's
// loop) is brought together first, or it could arrive in parts.
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// a word of another CTA's shared memory (shared::cluster address)
__device__ __forceinline__ void store_cluster(uint32_t cluster_addr, int v) {
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// The end of a pair of which either CTA aborted; the even CTA's part (the odd one waits at the cluster
// barrier behind it).  Every load of the pair counts on the even CTA's barriers, full(stage), which it
// armed for its own `mine` fills with both CTAs' bytes.  Where only one of the two issued a fill, the
// odd CTA's bytes are made up for: counted as there, or armed for alone once the stage's fill before is
// complete.
template <typename F>
__device__ __forceinline__ void drain_pair_loads(int mine, int odd, int stages, uint32_t odd_bytes, F&& full, int* err,
                                                 int code) {
    volatile int gave_up = 0;
    for (int j = max(0, mine - stages); j < max(mine, odd); ++j) {
        const uint32_t bar = full(j % stages);
        if (j >= mine) mbar_expect_tx(bar, odd_bytes);
        else if (j >= odd)
            asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(odd_bytes) : "memory");
        if (!mbar_wait(bar, (uint32_t)(j / stages) & 1, &gave_up, err, code)) return;
    }
}

// arrive on an mbarrier of another CTA of the cluster (shared::cluster address)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// 2D TMA load into this CTA's shared memory whose completion is counted on `bar`, an
// mbarrier of either CTA of the pair (shared::cluster address); no multicast
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// D (TMEM of both CTAs, 128 rows each) += A (128 rows in each CTA) * B (N/2 rows in each CTA)
__device__ __forceinline__ void tc_mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum)
        : "memory");
}

// tc_mma_pair issued by the elected lane of a converged warp (see tc_mma_elect)
__device__ __forceinline__ void tc_mma_pair_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                                  uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accum)
        : "memory");
}

// tc_commit_pair by the elected lane (the lane that issued the MMAs of tc_mma_pair_elect)
__device__ __forceinline__ void tc_commit_pair_elect(uint32_t bar, uint16_t cta_mask) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
        ::"r"(bar), "h"(cta_mask)
        : "memory");
}

// completion of this thread's earlier pair MMAs arrives once on the mbarrier at the same
// shared-memory offset in every CTA of `cta_mask`
__device__ __forceinline__ void tc_commit_pair(uint32_t bar, uint16_t cta_mask) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(cta_mask)
                 : "memory");
}

// One k-step of the block-scaled GEMM, issued by the elected lane of a converged warp: the scales of
// 256 columns of A and B from shared memory to TMEM (tcgen05.cp 32x128b.warpx4: 32 rows x 16 bytes to
// 4 columns of lanes 0..31, repeated in the other lane quarters), then
//   D (TMEM) += (A * its scales) (B * its scales)
// in four MMAs of K = 64, which find the scales of one 128-column group after the other, in the low
// and the high halves of its words, and a commit to `bar`.  NBLK: 128-row scale blocks of B; its two
// groups lie 512 bytes apart in shared memory, its blocks 1024.  sfb_rows: the TMEM word of B's
// first row.  CG 2: issued in the even CTA of a pair, whose CTAs each hold 128 rows of A, half the
// rows of B, the scales of their own rows of A and those of all rows of B; the commit reaches both.
// All in one statement: with an elect.sync for each instruction a step took 330 clocks to issue.
template <int CG, int NBLK>
__device__ __forceinline__ void tc_mxf4_step_elect(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint64_t sa_desc,
                                                   uint64_t sb_desc, uint32_t sfa, uint32_t sfb, uint32_t sfb_rows,
                                                   uint32_t idesc_lo, uint32_t idesc_hi, uint32_t accum, uint32_t bar) {
    static_assert((CG == 1 && NBLK == 1) || (CG == 2 && (NBLK == 1 || NBLK == 2)), "");
    if constexpr (CG == 1 && NBLK == 1)
        asm volatile(
            "{\n\t.reg .pred e, p, q;\n\t.reg .b32 t, u;\n\t.reg .b64 x, y;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %10, 0;\n\t"
            "setp.eq.b32 q, 0, 0;\n\t"
            "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%5], %3;\n\t"
            "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%6], %4;\n\t"
            "add.s32 t, %5, 4;\n\t"
            "add.s64 x, %3, 32;\n\t"
            "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [t], x;\n\t"
            "add.s32 t, %6, 4;\n\t"
            "add.s64 x, %4, 32;\n\t"
            "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [t], x;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %8, [%5], [%7], p;\n\t"
            "add.s64 x, %1, 2;\n\tadd.s64 y, %2, 2;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %9, [%5], [%7], q;\n\t"
            "add.s64 x, %1, 4;\n\tadd.s64 y, %2, 4;\n\t"
            "add.s32 t, %5, 4;\n\tadd.s32 u, %7, 4;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %8, [t], [u], q;\n\t"
            "add.s64 x, %1, 6;\n\tadd.s64 y, %2, 6;\n\t"
            "add.s32 t, %5, 4;\n\tadd.s32 u, %7, 4;\n\t"
            "@e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %9, [t], [u], q;\n\t"
            "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%11];\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "l"(sa_desc), "l"(sb_desc), "r"(sfa), "r"(sfb), "r"(sfb_rows), "r"(idesc_lo),
              "r"(idesc_hi), "r"(accum), "r"(bar)
            : "memory");
    else if constexpr (CG == 2 && NBLK == 1)
        asm volatile(
            "{\n\t.reg .pred e, p, q;\n\t.reg .b32 t, u;\n\t.reg .b64 x, y;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %10, 0;\n\t"
            "setp.eq.b32 q, 0, 0;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%5], %3;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%6], %4;\n\t"
            "add.s32 t, %5, 4;\n\t"
            "add.s64 x, %3, 32;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [t], x;\n\t"
            "add.s32 t, %6, 4;\n\t"
            "add.s64 x, %4, 32;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [t], x;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %8, [%5], [%7], p;\n\t"
            "add.s64 x, %1, 2;\n\tadd.s64 y, %2, 2;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %9, [%5], [%7], q;\n\t"
            "add.s64 x, %1, 4;\n\tadd.s64 y, %2, 4;\n\t"
            "add.s32 t, %5, 4;\n\tadd.s32 u, %7, 4;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %8, [t], [u], q;\n\t"
            "add.s64 x, %1, 6;\n\tadd.s64 y, %2, 6;\n\t"
            "add.s32 t, %5, 4;\n\tadd.s32 u, %7, 4;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %9, [t], [u], q;\n\t"
            "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%11], %12;\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "l"(sa_desc), "l"(sb_desc), "r"(sfa), "r"(sfb), "r"(sfb_rows), "r"(idesc_lo),
              "r"(idesc_hi), "r"(accum), "r"(bar), "h"((uint16_t)3)
            : "memory");
    else if constexpr (CG == 2 && NBLK == 2)
        asm volatile(
            "{\n\t.reg .pred e, p, q;\n\t.reg .b32 t, u;\n\t.reg .b64 x, y;\n\t"
            "elect.sync _|e, 0xffffffff;\n\t"
            "setp.ne.b32 p, %10, 0;\n\t"
            "setp.eq.b32 q, 0, 0;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%5], %3;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%6], %4;\n\t"
            "add.s32 t, %6, 4;\n\t"
            "add.s64 x, %4, 64;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [t], x;\n\t"
            "add.s32 t, %5, 4;\n\t"
            "add.s64 x, %3, 32;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [t], x;\n\t"
            "add.s32 t, %6, 8;\n\t"
            "add.s64 x, %4, 32;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [t], x;\n\t"
            "add.s32 t, %6, 12;\n\t"
            "add.s64 x, %4, 96;\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [t], x;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %8, [%5], [%7], p;\n\t"
            "add.s64 x, %1, 2;\n\tadd.s64 y, %2, 2;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %9, [%5], [%7], q;\n\t"
            "add.s64 x, %1, 4;\n\tadd.s64 y, %2, 4;\n\t"
            "add.s32 t, %5, 4;\n\tadd.s32 u, %7, 8;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %8, [t], [u], q;\n\t"
            "add.s64 x, %1, 6;\n\tadd.s64 y, %2, 6;\n\t"
            "add.s32 t, %5, 4;\n\tadd.s32 u, %7, 8;\n\t"
            "@e tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], x, y, %9, [t], [u], q;\n\t"
            "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%11], %12;\n\t}"
            ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "l"(sa_desc), "l"(sb_desc), "r"(sfa), "r"(sfb), "r"(sfb_rows), "r"(idesc_lo),
              "r"(idesc_hi), "r"(accum), "r"(bar), "h"((uint16_t)3)
            : "memory");
}

// untiled bulk copy (16-byte aligned, a multiple of 16 bytes) counted on an mbarrier of this CTA
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
                 : "memory");
}

// cuTensorMapEncodeTiled through the runtime's driver entry point (no libcuda link)
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();

}  // namespace tc
}  // namespace vdit
