// Linear on 4-bit microscaled operands (mx.cuh) on the block-scaled tcgen05 MMA:
//   out[m, n] = bf16( sum over blocks b of 2^(sa[m,b] + sw[n,b]) * sum_{j < 32} a[m,b,j] w[n,b,j] + bias[n] )
//
// Persistent CTA pairs (clusters of two, cta_group::2) walk 256 x BN output tiles, or, for few
// tiles, single CTAs 128 x BN ones.  A k-step is 256 elements (128 bytes) of 128 rows of a and of
// the CTA's share of the BN rows of w, and their scales.  Warp roles in each CTA:
//   warp 0      TMA producer: the codes as 128-byte-wide boxes (128-byte swizzle, K-major), the
//               scales in the 512-byte blocks they are stored in, into a ring; a pair's loads
//               all complete on the even CTA's stage barrier
//   warp 1      MMA issuer (even CTA): copies the k-step's scales from shared memory to the ring
//               stage's TMEM columns (tcgen05.cp), then four 64-deep MMAs
//   warps 2..9  epilogue: bias, rounding and TMA stores of one accumulator while the MMAs of the
//               next tile fill the other
// A k-step's MMAs take 512 clocks at the full rate, whatever its element type, so the issuer has to
// get through a k-step's waits, copies and MMAs in less; the notes in its loop say what that took.
// Two 256-column accumulators and 5 stages x 24 columns of scales do not fit TMEM's 512, so the
// second accumulator starts 120 columns early and each tile's epilogue empties the shared columns
// first, before the next tile's MMAs start.
//
// Every mbarrier wait is bounded; a wait that runs out records an error in g_mxlinear_error,
// raises the CTA abort flag and the CTA skips to its teardown (cluster barrier, TMEM always freed).
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

constexpr int BM = 128;                 // rows per CTA
constexpr int BK = 256;                 // elements of a k-step: 128 bytes of codes
constexpr int EPI_WARPS = 8;             // two for each quarter of the 128 TMEM lanes
constexpr int kThreads = (2 + EPI_WARPS) * 32;
constexpr int kErr = 0x4D58;            // "MX": a bounded wait of the linear ran out
constexpr int kScaleBlock = 512;        // 128 rows x 4 scales
constexpr int kMaxSize = INT32_MAX - 1024;   // tile coordinates stay int32

template <int CG, int BN>
struct __align__(1024) Smem {
    static constexpr int NBLK = BN > 128 ? 2 : 1;           // 128-row scale blocks a tile of w touches
    static constexpr int NST = BN > 128 ? 5 : 6;
    uint8_t a[NST][BM * 128];
    uint8_t w[NST][BN / CG * 128];                          // this CTA's share of the weight tile
    uint8_t x[EPI_WARPS][32 * 128];                         // a 32-row x 64-column box a warp
    uint8_t sa[NST][2 * kScaleBlock];
    uint8_t sw[NST][NBLK][2 * kScaleBlock];                 // the scales of the whole weight tile
    float bias[EPI_WARPS][BN];
    uint64_t full[NST], empty[NST], acc_full[2], acc_empty[2], shared_empty;
    uint64_t drained;                                       // after an abort: every MMA issued has ended
    uint32_t tmem_slot;
    int abort_flag;
    int peer_fills;                                         // after an abort: the loads that the pair's other CTA issued
};

struct Args {
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

template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 1) tma_load_2d(dst, map, x, y, bar);
    else tma_load_2d_pair(dst, map, x, y, mapa_shared(bar, 0));
}
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (CG == 1) tc_commit_elect(bar);
    else tc_commit_pair_elect(bar, 0x3);
}
// One arrival on the MMA issuer's barrier (in the even CTA of a pair), after the thread's TMEM loads
// have completed.  Nothing in memory is handed over, so the odd CTA's arrival is a relaxed one: a
// release to the cluster took ~1000 clocks here, between a tile's last MMA and the next one's first.
template <int CG>
__device__ __forceinline__ void arrive_issuer(uint32_t bar, uint32_t rank) {
    if (CG == 1 || rank == 0) mbar_arrive(bar);
    else
        asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(mapa_shared(bar, 0)) : "memory");
}

template <int CG, int BN>
__global__ void __launch_bounds__(kThreads, 1) linear_kernel(const __grid_constant__ CUtensorMap tmA,
                                                             const __grid_constant__ CUtensorMap tmW,
                                                             const __grid_constant__ CUtensorMap tmSA,
                                                             const __grid_constant__ CUtensorMap tmSW,
                                                             const __grid_constant__ CUtensorMap tmO,
                                                             const __grid_constant__ Args p) {
    extern __shared__ uint8_t raw[];
    using SM = Smem<CG, BN>;
    constexpr int NST = SM::NST, NBLK = SM::NBLK, BNC = BN / CG;
    constexpr uint32_t kStageBytes = CG * ((BM + BNC) * 128 + (1 + NBLK) * 2 * kScaleBlock);
    constexpr uint32_t kSfCols = 8 + 8 * NBLK;              // TMEM columns of one k-step's scales
    constexpr uint32_t kTmemCols = 512;
    constexpr uint32_t kSf0 = kTmemCols - NST * kSfCols;    // a set of scales per ring stage, at the end
    constexpr uint32_t kAcc1 = 2 * BN <= kSf0 ? BN : kSf0 - BN;
    constexpr bool kShared = kAcc1 < BN;                    // the accumulators share columns [kAcc1, BN)
    static_assert(!kShared || BN - kAcc1 <= 128, "the shared columns are the first part each epilogue warp reads");
    SM& sm = *reinterpret_cast<SM*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    // through a shuffle the warp index is uniform to the compiler, which then keeps the MMA
    // operands of its branch in uniform registers
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = CG == 1 ? 0 : cluster_rank();
    const int unit = blockIdx.x / CG, nunits = gridDim.x / CG;
    volatile int* abort_flag = &sm.abort_flag;
    // rows, columns, steps and scales past the operands read zeros (the tensor maps' fill)
    const int tiles_m = (int)((p.m + CG * BM - 1) / (CG * BM)), tiles_n = (p.n + BN - 1) / BN;
    const int ntiles = tiles_m * tiles_n;
    const int nk = (p.k + BK - 1) / BK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbar_init(smem_u32(&sm.full[s]), 1);
            mbar_init(smem_u32(&sm.empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&sm.acc_full[b]), 1);
            mbar_init(smem_u32(&sm.acc_empty[b]), CG * EPI_WARPS);
        }
        mbar_init(smem_u32(&sm.shared_empty), CG * EPI_WARPS);
        mbar_init(smem_u32(&sm.drained), 1);
        sm.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (const CUtensorMap* map : {&tmA, &tmW, &tmSA, &tmSW, &tmO})
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
    }
    if (warp == 1) {
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(smem_u32(&sm.tmem_slot)), "r"(kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                         ::"r"(smem_u32(&sm.tmem_slot)), "r"(kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        }
        tc_fence_before();
    }
    __syncthreads();
    if (CG == 2) cluster_sync();     // the peer's barriers are initialised before anyone signals them
    tc_fence_after();
    // all 512 columns are this CTA's, so they start at 0: a constant, as MMA operands from shared
    // memory would pass through vector registers
    constexpr uint32_t tmem = 0;
    int fills = 0;                                          // producer: loads issued into the ring

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (every CTA)
        if (lane == 0) {
            // a is written, when launched beside its writer.  That one lets this kernel start only after
            // its own wait, so all older kernels are complete: the epilogue reads the bias without a wait.
            asm volatile("griddepcontrol.wait;" ::: "memory");
            int& it = fills;
            bool ok = true;
            for (int t = unit; ok && t < ntiles; t += nunits) {
                int tm, tn;
                tile_coords(t, tiles_m, tiles_n, tm, tn);
                const int rb = tm * CG + (int)rank;         // this CTA's rows of a, in blocks of 128
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int s = it % NST;
                    if (it >= NST &&
                        !mbar_wait(smem_u32(&sm.empty[s]), ((it / NST) - 1) & 1, abort_flag, &g_mxlinear_error, kErr)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = smem_u32(&sm.full[s]);
                    if (rank == 0) mbar_expect_tx(bar, kStageBytes);
                    load_box<CG>(smem_u32(sm.sa[s]), &tmSA, kb * 256, rb, bar);
                    load_box<CG>(smem_u32(sm.sw[s]), &tmSW, kb * 256, tn * BN / 128, bar);
                    load_box<CG>(smem_u32(sm.a[s]), &tmA, kb * 128, rb * BM, bar);
                    load_box<CG>(smem_u32(sm.w[s]), &tmW, kb * 128, tn * BN + (int)rank * BNC, bar);
                }
            }
            // every commit on this CTA's stages has arrived before it leaves: the tensor core delivers them to
            // both CTAs of a pair by itself, which the cluster barrier at the end does not wait for
            for (int j = max(0, it - NST); ok && j < it; ++j)
                ok = mbar_wait(smem_u32(&sm.empty[j % NST]), (j / NST) & 1, abort_flag, &g_mxlinear_error, kErr);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer (even CTA)
        // the whole warp runs the loop, the elected lane issues, with descriptors as bases plus
        // stage and k offsets so they stay in uniform registers
        if (rank == 0) {
            const uint64_t ad0 = make_desc(smem_u32(sm.a[0]), 16, 1024, kSw128);
            const uint64_t wd0 = make_desc(smem_u32(sm.w[0]), 16, 1024, kSw128);
            const uint64_t sad0 = make_desc(smem_u32(sm.sa[0]), 16, 128, 0);
            const uint64_t swd0 = make_desc(smem_u32(sm.sw[0]), 16, 128, 0);
            auto wait = [&](uint32_t bar, uint32_t parity) {
                return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, &g_mxlinear_error, kErr));
            };
            int it = 0, lt = 0;
            bool ok = true, early = false;                  // early: the next step's data has been seen to be there
            for (int t = unit; ok && t < ntiles; t += nunits, ++lt) {
                const int buf = lt & 1;
                int tm, tn;
                tile_coords(t, tiles_m, tiles_n, tm, tn);
                const uint32_t shift = (uint32_t)(tn * BN % 128) / 32;   // scale columns before the tile's first row
                if (lt >= 2 && !wait(smem_u32(&sm.acc_empty[buf]), ((lt >> 1) - 1) & 1)) break;
                if (kShared && lt >= 1 && !wait(smem_u32(&sm.shared_empty), (lt - 1) & 1)) break;
                tc_fence_after();
                const uint32_t acc = tmem + buf * kAcc1;
                for (int kb = 0; kb < nk; ++kb, ++it) {
                    const int s = it % NST;
                    if (!early && !wait(smem_u32(&sm.full[s]), (it / NST) & 1)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    // ask for the next step before this one is issued: the answer takes ~200 clocks
                    const int s1 = (it + 1) % NST;
                    const bool next = mbar_test(smem_u32(&sm.full[s1]), ((it + 1) / NST) & 1);
                    const uint32_t sfa = tmem + kSf0 + s * kSfCols, sfw = sfa + 8;
                    // all four MMAs also in a partial last step, where they add zeros: with a branch
                    // around each they took twice as long to issue
                    tc_mxf4_step_elect<CG, NBLK>(
                        acc, ad0 + (uint64_t)(s * (int)(sizeof(sm.a[0]) >> 4)),
                        wd0 + (uint64_t)(s * (int)(sizeof(sm.w[0]) >> 4)),
                        sad0 + (uint64_t)(s * (int)(sizeof(sm.sa[0]) >> 4)),
                        swd0 + (uint64_t)(s * (int)(sizeof(sm.sw[0]) >> 4)), sfa, sfw, sfw + shift,
                        make_idesc_mxf4(CG * BM, BN, 0), make_idesc_mxf4(CG * BM, BN, 2), (uint32_t)(kb > 0),
                        smem_u32(&sm.empty[s]));
                    early = __all_sync(0xffffffffu, next);
                }
                if (ok) commit<CG>(smem_u32(&sm.acc_full[buf]));
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue (every CTA)
        // Two warps share each lane quarter (32 rows), one taking the even, one the odd 64-column
        // parts of a tile.  A warp first reads its parts into registers, which frees the accumulator,
        // then turns one after another into bf16 in its staging box (128-byte swizzle), which one
        // lane stores; a second box a warp would cost a ring stage (95 against 86 us for
        // 16384 x 7680 x 1536).  The map clips rows past m and columns past n.  The tile's bias is
        // in shared memory before its accumulator is ready.
        constexpr int PARTS = (BN / 64 + 1) / 2;            // parts of a warp, at most
        const int ew = warp - 2, quarter = warp & 3, odd = ew >> 2;
        const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
        float* bias = sm.bias[ew];
        uint8_t* box = sm.x[ew];
        int lt = 0;
        for (int t = unit; t < ntiles; t += nunits, ++lt) {
            const int buf = lt & 1;
            int tm, tn;
            tile_coords(t, tiles_m, tiles_n, tm, tn);
            const int64_t row0 = ((int64_t)tm * CG + rank) * BM + quarter * 32;
            const int col0 = tn * BN;
            __syncwarp();                                   // every lane has read the last tile's bias
            for (int c = lane * 8; c < BN; c += 256) {      // n is a multiple of 8
                float bv[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                if (p.bias && col0 + c < p.n) load8_nc(p.bias + col0 + c, bv);
                *reinterpret_cast<float4*>(bias + c) = make_float4(bv[0], bv[1], bv[2], bv[3]);
                *reinterpret_cast<float4*>(bias + c + 4) = make_float4(bv[4], bv[5], bv[6], bv[7]);
            }
            __syncwarp();
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.acc_full[buf]), (lt >> 1) & 1, abort_flag,
                                                   &g_mxlinear_error, kErr)))
                break;
            tc_fence_after();
            // the first accumulator's last two parts and the second one's first two hold the columns
            // both share: each warp reads its one of them first and says so
            const bool reversed = kShared && buf == 0;
            float v[PARTS][64];
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                const int c = 2 * (reversed ? PARTS - 1 - i : i) + odd;
                if (c < BN / 64) {
                    tmem_ld32(tmem + buf * kAcc1 + c * 64 + lane_off, v[i]);
                    tmem_ld32(tmem + buf * kAcc1 + c * 64 + 32 + lane_off, v[i] + 32);
                    tmem_wait_ld();
                }
                if (i == PARTS - 1 || (kShared && i == 0)) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_issuer<CG>(smem_u32(i == PARTS - 1 ? &sm.acc_empty[buf] : &sm.shared_empty), rank);
                }
            }
            if (row0 >= p.m) continue;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                const int c = 2 * (reversed ? PARTS - 1 - i : i) + odd;
                if (c >= BN / 64 || col0 + c * 64 >= p.n) continue;
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const float4 b = *reinterpret_cast<const float4*>(bias + c * 64 + q * 4);
                    v[i][q * 4] += b.x;
                    v[i][q * 4 + 1] += b.y;
                    v[i][q * 4 + 2] += b.z;
                    v[i][q * 4 + 3] += b.w;
                }
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    *reinterpret_cast<uint4*>(box + lane * 128 + ((q ^ (lane & 7)) << 4)) = pack8(v[i] + q * 8);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(&tmO, smem_u32(box), col0 + c * 64, (int)row0);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }

    tc_fence_before();
    __syncthreads();
    if (CG == 2) {
        // an abort is the pair's: the peer need not wait its own limit out
        if (threadIdx.x == 0 && *abort_flag) store_cluster(mapa_shared(smem_u32(&sm.abort_flag), rank ^ 1), 1);
        cluster_sync();              // no CTA leaves while its peer's MMAs or arrivals may still touch it
    }
    if (*abort_flag) {
        // a wait ran out: the loads and MMAs still in flight end before any CTA of them does
        if (CG == 2) {
            if (threadIdx.x == 0) store_cluster(mapa_shared(smem_u32(&sm.peer_fills), rank ^ 1), fills);
            cluster_sync();
        }
        auto full = [&](int s) { return smem_u32(&sm.full[s]); };
        if (rank == 0 && warp == 1) {
            volatile int gave_up = 0;
            if constexpr (CG == 1) tc_commit_elect(smem_u32(&sm.drained));
            else tc_commit_pair_elect(smem_u32(&sm.drained), 0x1);
            mbar_wait(smem_u32(&sm.drained), 0, &gave_up, &g_mxlinear_error, kErr);
        } else if (rank == 0 && threadIdx.x == 0) {
            if (CG == 1) drain_loads(0, fills, NST, full, &g_mxlinear_error, kErr);
            else drain_pair_loads(fills, sm.peer_fills, NST, kStageBytes / 2, full, &g_mxlinear_error, kErr);
        }
        __syncthreads();
        if (CG == 2) cluster_sync();
    }
    if (warp == 1) {
        tc_fence_after();
        if constexpr (CG == 1)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sm.tmem_slot), "r"(kTmemCols));
        else
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(sm.tmem_slot), "r"(kTmemCols));
    }
}

bool make_map(CUtensorMap* map, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* base, int64_t rows,
              int64_t cols, int64_t ld_bytes, int box_rows, int box_cols) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld_bytes};
    cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    cuuint32_t es[2] = {1, 1};
    return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// codes of a [rows, k] operand: 128-byte-wide boxes
bool code_map(CUtensorMap* map, const void* codes, int64_t rows, int k, int box_rows) {
    return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, codes, rows, k / 2, k / 2, box_rows, 128);
}
// its scales as rows of 512-byte blocks: two blocks (one k-step) of box_blocks block rows
bool scale_map(CUtensorMap* map, const void* scales, int64_t rows, int k, int box_blocks) {
    const int64_t words = (int64_t)scale_col_groups(k) * (kScaleBlock / 4);
    return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, CU_TENSOR_MAP_SWIZZLE_NONE, scales, scale_row_blocks(rows), words,
                    words * 4, box_blocks, 2 * kScaleBlock / 4);
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

struct Call {
    const void *a, *as, *w, *ws;
    CUtensorMap out;
    Args p;
    int dev, sms;
    bool after_quantize;
    cudaStream_t stream;
};

template <int CG, int BN>
int launch(const Call& c) {
    // units (CTAs or pairs) resident at once, asked once per device; 0: not asked yet
    static std::atomic<int> resident[kMaxDevices];
    const Args& p = c.p;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Smem<CG, BN>) + 1024;
    cfg.stream = c.stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int units = resident[c.dev].load(std::memory_order_acquire);
    if (units == 0) {
        cudaError_t e = cudaFuncSetAttribute(linear_kernel<CG, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)cfg.dynamicSmemBytes);
        units = c.sms / CG;
        if (e == cudaSuccess && CG == 2) {
            cfg.gridDim = dim3(CG * units);
            e = cudaOccupancyMaxActiveClusters(&units, linear_kernel<CG, BN>, &cfg);
        }
        if (e != cudaSuccess || units <= 0) {
            record_cuda_error(e != cudaSuccess ? e : cudaErrorInvalidConfiguration);
            return VDIT_ERR_LAUNCH;
        }
        resident[c.dev].store(units, std::memory_order_release);
    }
    CUtensorMap ma, mw, msa, msw;
    if (!code_map(&ma, c.a, p.m, p.k, BM) || !code_map(&mw, c.w, p.n, p.k, BN / CG) ||
        !scale_map(&msa, c.as, p.m, p.k, 1) || !scale_map(&msw, c.ws, p.n, p.k, Smem<CG, BN>::NBLK))
        return VDIT_ERR_DRIVER;
    const int64_t tiles = ((p.m + CG * BM - 1) / (CG * BM)) * ((p.n + BN - 1) / BN);
    if (tiles > INT32_MAX / 2) return VDIT_ERR_UNSUPPORTED;
    cfg.gridDim = dim3((unsigned)(CG * std::min<int64_t>(tiles, units)));
    cfg.numAttrs = c.after_quantize ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_kernel<CG, BN>, ma, mw, msa, msw, c.out, p);
    if (e != cudaSuccess) {
        record_cuda_error(e);
        return VDIT_ERR_LAUNCH;
    }
    count_launches(1);
    return check_launch();
}

// Tile for an [m, n] output: of the pairs' widths and the single CTA's 64 columns the one with
// the least estimated time, rounds of tiles over the GPU x the time of a tile (whose ratios hardly depend
// on k).  Product alone, us on 256 / 192 / 128 / 64 columns, * the one picked:
//   k = 1536   128 x 1536 7.5 / 7.0 / 6.3 / 5.1*, 2048 x 1536 9.0 / 8.5* / 9.3 / 10.0,
//              4101 x 1536 11.8 / 11.2* / 11.6 / 16.0, 4101 x 7680 27.9* / 31.5 / 36.7 / 59.9
//   k = 3840   128 x 1536 10.5 / 10.2 / 9.4 / 8.2*, 2048 x 1536 12.0 / 11.4* / 14.6 / 17.3,
//              4632 x 1536 18.5* / 21.5 / 24.3 / 31.6, 16384 x 1536 42.4 / 44.0* / 59.2 / 101
//   k = 320    4101 x 7680 18.9* / 21.8 / 20.6 / 30.1, 4632 x 1536 9.2* / 9.8 / 9.1 / 9.9
int pick_tile(int64_t m, int n, int sms) {
    const int widths[4] = {256, 192, 128, 64};
    const double cost[4] = {1.0, 0.8, 0.6, 0.35};
    int best = 64;
    double best_t = 1e300;
    for (int i = 0; i < 4; ++i) {
        const int cg = widths[i] == 64 ? 1 : 2;
        const int64_t tiles = ((m + cg * BM - 1) / (cg * BM)) * ((n + widths[i] - 1) / widths[i]);
        const int64_t units = std::max(1, sms / cg);
        const double t = (double)((tiles + units - 1) / units) * cost[i];
        if (t < best_t) {
            best_t = t;
            best = widths[i];
        }
    }
    return best;
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

namespace vdit {
namespace mx {
namespace {

// The product of quantised rows; after_quantize: launched behind the kernel that writes a, beside whose
// end it starts.
int linear_codes(const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales, const void* bias,
                 void* out, int64_t ldo, int64_t m, int32_t n, int32_t k, bool after_quantize, cudaStream_t stream) {
    if (!a_codes || !a_scales || !w_codes || !w_scales || !out || m < 0 || n <= 0 || k <= 0 || ldo < n)
        return VDIT_ERR_ARG;
    if (n % 8 || k % kBlock || m > kMaxSize || n > kMaxSize || k > kMaxSize) return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(a_codes) || !aligned16(a_scales) || !aligned16(w_codes) || !aligned16(w_scales) || !aligned16(out) ||
        (bias && !aligned16(bias)) || ldo % 8)
        return VDIT_ERR_ALIGN;
    if (m == 0) return VDIT_OK;
    int sms;
    const int dev = current_device(&sms);
    if (dev < 0) return VDIT_ERR_UNSUPPORTED;
    Call c{a_codes, a_scales, w_codes, w_scales, {}, {static_cast<const __nv_bfloat16*>(bias), m, n, k}, dev, sms,
           after_quantize, stream};
    if (!make_map(&c.out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, out, m, n, ldo * 2, 32, 64))
        return VDIT_ERR_DRIVER;
    switch (pick_tile(m, n, sms)) {
        case 256: return launch<2, 256>(c);
        case 192: return launch<2, 192>(c);
        case 128: return launch<2, 128>(c);
        default: return launch<1, 64>(c);
    }
}

// ------------------------------------------------------------------ few dense rows
// Up to 4 rows of a read the weight once and quantise themselves on the way, in one launch: bound by
// latency.  A warp takes the four weight rows whose scales lie in one vector (r, r + 32, r + 64, r + 96
// of a 128-row block), a lane one block of 32 of each at a time; the first blocks are on their way
// before the CTA quantises the rows of a into shared memory.  Products of half a block are summed in
// f16 pairs, exactly: 8 products of at most 36, all multiples of 1/4, stay below 2^11 quarters.  Across
// blocks the sums are fp32; a block's sum takes the smaller of its two scales first, so that the
// product overflows only where the result does.
// One and two rows, graph replays with weights beyond L2, no bias, here / by the quantiser and the MMA kernel, us:
// 7680 x 1536 5.8, 7.0 / 7.6, 1536 x 1536 3.7, 4.5 / 5.4, 16384 x 4096 15, 20 / 21.  Three and four rows are
// the slower ones on the GPU, but a launch less is host time where calls follow one another from Python;
// graph (calls), here / there: 1536 x 640 4.3 (9) / 4.5 (13), 1536 x 2048 6.2 (9) / 6.1 (13), 7680 x 1536 12.4 (14) /
// 7.7 (13), 1536 x 2560 8.5 (10) / 6.9 (13), 1536 x 3840 11 (12) / 9.0 (13), 16384 x 4096 39 (41) / 21 (21).  So they
// come here up to k = 2048; the rule knows no n because the workspace's size does not.
constexpr int kFewRows = 4;
constexpr int kFewWide = 2048;
constexpr int kFewWarps = 8;
constexpr int64_t kFewElements = 65536;      // of a, rows rounded up: 136 KB of shared memory
constexpr int kFewSmem = (int)(kFewElements * 2 + kFewElements / kBlock * 4);

int few_rounded(int64_t m) { return m <= 2 ? (int)m : 4; }
bool few_rows(int64_t m, int k) {
    return m <= kFewRows && (m <= 2 || k <= kFewWide) && (int64_t)few_rounded(m) * k <= kFewElements;
}

struct FewArgs {
    const void* x;
    int64_t ldx;
    const uint8_t *w, *ws;
    const __nv_bfloat16* bias;
    __nv_bfloat16* out;
    int64_t ldo;
    int m, n, k;
};

__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 pair(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// the smaller and the larger of two scales; a NaN stays one
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// MT: rows of a, rounded up to a power of two (the rows past m are zeros)
template <int T, int MT>
__global__ void __launch_bounds__(kFewWarps * 32) few_rows_kernel(const __grid_constant__ FewArgs p) {
    extern __shared__ __align__(16) uint8_t few[];
    uint4* xs = reinterpret_cast<uint4*>(few);                          // [MT][blocks][4] chunks of 8 elements, f16
    const int blocks = p.k / kBlock;
    float* xscale = reinterpret_cast<float*>(few + (size_t)MT * p.k * 2);   // [MT][blocks]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int groups = scale_col_groups(p.k);
    const int task = blockIdx.x * kFewWarps + warp;
    const int row0 = (task >> 5) * 128 + (task & 31);
    const bool live = row0 < p.n;
    const uint8_t* scales = p.ws + (int64_t)(task >> 5) * groups * 512 + (task & 31) * 16;
    uint4 c[4], s;
    auto fetch = [&](int b) {                               // block b of the four rows
#pragma unroll
        for (int r = 0; r < 4; ++r)
            c[r] = live && b < blocks && row0 + 32 * r < p.n
                       ? __ldg(reinterpret_cast<const uint4*>(p.w + (int64_t)(row0 + 32 * r) * (p.k / 2)) + b)
                       : make_uint4(0, 0, 0, 0);
        s = live && b < blocks ? __ldg(reinterpret_cast<const uint4*>(scales + (b >> 2) * 512)) : make_uint4(0, 0, 0, 0);
    };
    fetch(lane);

    // quantise a: half a block a thread, two of them at a time; the 16-byte chunks of a block are
    // rotated so that 8 lanes reading the same chunk of 8 blocks meet different banks
    const int per_row = p.k / 16, halves = MT * per_row;
    for (int i0 = threadIdx.x; i0 < halves; i0 += 2 * kFewWarps * 32) {
        Half<T> v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = i0 + u * kFewWarps * 32, row = i / per_row;
            if (i < halves && row < p.m)
                v[u].load(static_cast<const typename Elem<T>::type*>(p.x) + row * p.ldx + (i - row * per_row) * 16);
            else
                v[u].zero();
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = i0 + u * kFewWarps * 32;
            if (i >= halves) break;                         // both threads of a block
            const int at = i >> 1, j = (i & 1) * 2;         // block (of all rows) and first chunk
            const unsigned two = 3u << (threadIdx.x & 30);
            uint32_t top = v[u].amax();
            top = max(top, __shfl_xor_sync(two, top, 1));
            const uint32_t e = scale_byte<4>(top);
            const float inv = scale_inverse(e);
            uint32_t h[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float2 y = fmul2(v[u].pair(q), inv);
                h[q] = e == 255 ? 0u : bits(__floats2half2_rn(round_e2m1(y.x), round_e2m1(y.y)));
            }
            const int turn = (at % blocks) >> 1 & 3;
            xs[at * 4 + (j ^ turn)] = make_uint4(h[0], h[1], h[2], h[3]);
            xs[at * 4 + ((j + 1) ^ turn)] = make_uint4(h[4], h[5], h[6], h[7]);
            if (j == 0) xscale[at] = scale_value(e);
        }
    }
    __syncthreads();
    if (!live) return;

    float acc[4][MT];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[r][i] = 0.f;
    for (int b0 = 0; b0 < blocks; b0 += 32) {
        const int b = b0 + lane;
        __half2 w[4][16];
        float sc[4];
        const uint32_t word[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            decode8_e2m1(c[r].x, w[r]);
            decode8_e2m1(c[r].y, w[r] + 4);
            decode8_e2m1(c[r].z, w[r] + 8);
            decode8_e2m1(c[r].w, w[r] + 12);
            sc[r] = scale_value((word[r] >> (8 * (b & 3))) & 255u);
        }
        if (b0 + 32 < blocks) fetch(b + 32);
        if (b < blocks) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                __half2 x[16];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 u = xs[(i * blocks + b) * 4 + (j ^ (b >> 1 & 3))];
                    x[4 * j] = pair(u.x);
                    x[4 * j + 1] = pair(u.y);
                    x[4 * j + 2] = pair(u.z);
                    x[4 * j + 3] = pair(u.w);
                }
                const float e = xscale[i * blocks + b];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    __half2 h0 = __hmul2(w[r][0], x[0]), h1 = __hmul2(w[r][8], x[8]);
#pragma unroll
                    for (int j = 1; j < 8; ++j) {
                        h0 = __hfma2(w[r][j], x[j], h0);
                        h1 = __hfma2(w[r][8 + j], x[8 + j], h1);
                    }
                    const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
                    acc[r][i] = fmaf(((f0.x + f0.y) + (f1.x + f1.y)) * min_nan(sc[r], e), max_nan(sc[r], e), acc[r][i]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if (i >= p.m) break;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = warp_sum(acc[r][i]);
            const int col = row0 + 32 * r;
            if (lane == r && col < p.n) p.out[i * p.ldo + col] = f2bf(v + (p.bias ? bf2f(p.bias[col]) : 0.f));
        }
    }
}

template <int T, int MT>
int launch_few(const FewArgs& p, int dev, cudaStream_t s) {
    static std::atomic<bool> ready[kMaxDevices];            // the largest shared memory size is set, per device
    const size_t smem = (size_t)MT * p.k * 2 + (size_t)MT * (p.k / kBlock) * 4;
    if (smem > 48 * 1024 && !ready[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(few_rows_kernel<T, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   kFewSmem);
        if (e != cudaSuccess) {
            record_cuda_error(e);
            return VDIT_ERR_LAUNCH;
        }
        ready[dev].store(true, std::memory_order_release);
    }
    const int tasks = (p.n + 127) / 128 * 32;
    few_rows_kernel<T, MT><<<(tasks + kFewWarps - 1) / kFewWarps, kFewWarps * 32, smem, s>>>(p);
    count_launches(1);
    return check_launch();
}

template <int T>
int launch_few(const FewArgs& p, int dev, cudaStream_t s) {
    switch (few_rounded(p.m)) {
        case 1: return launch_few<T, 1>(p, dev, s);
        case 2: return launch_few<T, 2>(p, dev, s);
        default: return launch_few<T, 4>(p, dev, s);
    }
}

}  // namespace
}  // namespace mx
}  // namespace vdit

extern "C" int vdit_linear_mxfp4(const void* a_codes, const void* a_scales, const void* w_codes, const void* w_scales,
                                 const void* bias, void* out, int64_t ldo, int64_t m, int32_t n, int32_t k,
                                 vdit_stream_t stream) {
    return linear_codes(a_codes, a_scales, w_codes, w_scales, bias, out, ldo, m, n, k, false,
                        static_cast<cudaStream_t>(stream));
}

extern "C" size_t vdit_linear_mxfp4_dense_workspace_bytes(int64_t m, int32_t k) {
    if (m < 1 || k < 1 || few_rows(m, k)) return 0;
    return (size_t)m * (k / 2) + vdit_mxfp4_scale_bytes(m, k);
}

extern "C" int vdit_linear_mxfp4_dense(const void* x, int32_t x_type, int64_t ldx, const void* w_codes,
                                       const void* w_scales, const void* bias, void* out, int64_t ldo, int64_t m,
                                       int32_t n, int32_t k, void* workspace, size_t workspace_bytes,
                                       vdit_stream_t stream) {
    const int elem = x_type == VDIT_F32 ? 4 : x_type == VDIT_BF16 || x_type == VDIT_F16 ? 2 : 0;
    if (!elem || !x || !w_codes || !w_scales || !out || m < 0 || n <= 0 || k <= 0 || ldx < k || ldo < n)
        return VDIT_ERR_ARG;
    if (n % 8 || k % kBlock || m > kMaxSize || n > kMaxSize || k > kMaxSize) return VDIT_ERR_UNSUPPORTED;
    if (!aligned16(x) || (ldx * elem) % 16 || !aligned16(w_codes) || !aligned16(w_scales) || !aligned16(out) ||
        (bias && !aligned16(bias)) || ldo % 8)
        return VDIT_ERR_ALIGN;
    if (m == 0) return VDIT_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (few_rows(m, k)) {
        int sms;
        const int dev = current_device(&sms);
        if (dev < 0) return VDIT_ERR_UNSUPPORTED;
        const FewArgs p{x, ldx, static_cast<const uint8_t*>(w_codes), static_cast<const uint8_t*>(w_scales),
                        static_cast<const __nv_bfloat16*>(bias), static_cast<__nv_bfloat16*>(out), ldo, (int)m, n, k};
        if (x_type == VDIT_BF16) return launch_few<VDIT_BF16>(p, dev, s);
        if (x_type == VDIT_F16) return launch_few<VDIT_F16>(p, dev, s);
        return launch_few<VDIT_F32>(p, dev, s);
    }
    if (!workspace || workspace_bytes < vdit_linear_mxfp4_dense_workspace_bytes(m, k)) return VDIT_ERR_WORKSPACE;
    uint8_t* codes = static_cast<uint8_t*>(workspace);      // m * k / 2 bytes, a multiple of 16
    uint8_t* scales = codes + m * (int64_t)(k / 2);
    const int rc = vdit_mxfp4_quantize(x, x_type, ldx, m, k, codes, scales, stream);
    if (rc != VDIT_OK) return rc;
    return linear_codes(codes, scales, w_codes, w_scales, bias, out, ldo, m, n, k, true, s);
}
