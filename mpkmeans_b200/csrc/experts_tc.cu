/* experts_tc.cu -- the experts' products on tcgen05 (sm_100a).
 *
 * One persistent kernel for the product and its two gradients.  All three are
 * out[j][f] = sum_c A[f][c] B[j][c] for one expert, with f the output's contiguous
 * dimension (the 128 lanes of a TMEM accumulator) and j its rows (the columns):
 *
 *          f        j              c      A (128 f a CTA)        B (BN j)
 *   FWD    width    expert's rows  k      W_e, K-major           X rows, K-major
 *   GRADX  k        expert's rows  width  W_e, MN-major          GY rows, K-major
 *   GRADW  k        width          rows   X rows, MN-major       GY rows, MN-major
 *
 * so weights are always the wide operand's source, a short segment of rows costs
 * only a narrow tile, and every store of a warp runs along f.  The experts' row
 * counts are on the device only: each CTA scans them into shared memory and the
 * grid walks the tiles of all experts.  The launch has a cluster for every tile
 * there can be; a running cluster takes over the next one that has not started
 * (clusterlaunchcontrol), so uneven tiles spread evenly without a counter in
 * memory.  An element's sum is formed in one order whichever cluster does it.
 *
 *   warp 0      TMA producer: one 64-deep stage of A and B at a time; asks for the
 *               next tile as it starts one.
 *   warp 1      MMA issuer, whole contraction into one FP32 TMEM accumulator, two
 *               accumulators so that the next tile's MMAs overlap the epilogue.
 *   warps 2-9   epilogue: round to the output type, swap halves between lane
 *               pairs so that a lane holds two neighbouring f, store 4 bytes.
 *
 * Many rows an expert (PAIR): two CTAs on two SMs share each MMA (cta_group::2,
 * 256 f x up to 256 j).  Every CTA stages its 128 f of A and its half of the j's,
 * 32 KB for 256 x 256 x 64 products of the pair, half the operand traffic of
 * one-CTA 128 x 256 tiles.  The MMA is only as wide as the tile has rows (rounded
 * up to 32), so the last tile of a segment costs its share.  X comes sorted: the
 * caller copies gathered rows first.  (Gathering 128-byte pieces of rows inside
 * this kernel held 32768 x 4096 by 2048 at 0.80 ms with cp.async and 1.45 ms with
 * TMA's gather4, 45 ns an instruction; sorted rows take 0.45 ms and the copy
 * 0.06 ms.)
 *
 * Few rows an expert: one CTA, 128 f x 32 j, bound by reading W once, ten
 * stages of 20 KB in flight.  Gathered rows come by cp.async in warps 10-15, 16
 * bytes a copy, into the same swizzled layout.  Warp w fills ring slots w, w + 6,
 * ...: handing a stage to the tensor cores (proxy fence, arrive) waits for all
 * copies its warp has in flight, so stages overlap between warps, not within one;
 * and one warp sees every use of a slot, so it cannot be two phases behind the
 * slot's barrier, whose parity would then look like the next.
 *
 * Rows past a segment.  FWD and GRADX read whatever rows follow (the gather
 * writes zeros): a column of the accumulator depends on its own row only and those
 * columns are not stored.  GRADW contracts over the rows, so rows of the last stage
 * that are not the expert's must be zeros.  They come from a second tensor map of
 * the same matrix, three-dimensional with both outer strides one row: element
 * (c, y, z) is row y + z, y < 64.  A box of 64 rows from y = 64 - rem, z = end - 64
 * holds the segment's last rem rows, and the rest of it lies past y's bound, which
 * TMA fills with zeros.  (Segments that end before row 64 have no such z: gather4
 * with an index past the tensor for the other rows, 45 ns an instruction; all
 * tails that way made the gradient of 32 x 2048 x 4096 weights from 1200 rows
 * take 380 us.)
 */
#include "experts.cuh"
#include "mpkexperts.h"
#include "mpkmeans_debug.h"

#include <cudaTypedefs.h>

#include <mutex>

namespace mpk {
namespace {

/* Bounded waits that ran out in any product kernel of this device (MPK_DEV_* bits). */
__device__ int g_experts_status;

constexpr int BM = 128, BK = 64;
constexpr int kEpiWarps = 8;
constexpr int kGatherWarps = 6;
constexpr int BROWS = 32;                        /* rows of one K-major box of B */
constexpr int A_STAGE = BM * BK * 2;             /* 16 KB */
constexpr int BOX = 64 * 64 * 2;                 /* one 64 x 64 MN-major box */
constexpr int kSmemMax = 232448;
constexpr int kMisc = 1024 + 8 * (MPK_MAX_EXPERTS + 1);
constexpr int kInfo = 4;                         /* tiles between the producer and the epilogue */
constexpr int kAsk = 4;                          /* answers between asking for a tile and CTA 1's having read it */
constexpr int kMostTiles = 1 << 29;              /* more than any plan's; offsets that are none stay below it */
constexpr int kGroup = 8;                        /* row tiles that sweep the f tiles together */

template <bool PAIR, int BN>
struct Cfg {
    static constexpr int BL = PAIR ? BN / 2 : BN;              /* j's this CTA stages */
    static constexpr int FT = PAIR ? 2 * BM : BM;              /* f's of one tile */
    static constexpr int B_STAGE = BL * BK * 2;
    static constexpr int STAGE = A_STAGE + B_STAGE;
    static constexpr int RAW = (kSmemMax - kMisc) / STAGE;
    static constexpr int STAGES = RAW > 12 ? 12 : RAW;
    static constexpr int SMEM_BYTES = STAGES * STAGE + kMisc;
    static constexpr int TMEM_COLS = 2 * BN;
    static constexpr int HALF = BN / 2;                        /* columns an epilogue warp */
    static constexpr int CH = HALF < 32 ? HALF : 32;           /* columns of one TMEM load */
    static constexpr int THREADS = 64 + 32 * kEpiWarps + (PAIR ? 0 : 32 * kGatherWarps);
    static_assert(CH == 16 || CH == 32, "TMEM load width");
    static_assert(TMEM_COLS >= 32 && TMEM_COLS <= 512, "TMEM columns");
    static_assert(STAGE % 1024 == 0, "swizzle atoms");
};

/* One tile of one expert's output. */
struct Tile {
    int u;                      /* its index; -1: there are no more */
    int e;
    int r0, rows;               /* the expert's sorted rows */
    int j0, nj;                 /* first output row inside the expert, rows of this tile (0: an index past the tiles) */
    int wide;                   /* columns of the MMA */
    int f0;
    int nk;                     /* 64-deep contraction steps */
    int pad[3];
};
static_assert(sizeof(Tile) % 16 == 0, "moved in 16-byte words");

template <int STAGES>
struct EMisc {
    uint4 next[kAsk];              /* answers to ask_next (CTA 0) */
    int passed[kAsk];           /* the same as CTA 0 passes them to CTA 1 */
    Tile info[kInfo];           /* the tiles the producer has started */
    uint64_t full[STAGES], empty[STAGES], t_full[2], t_empty[2], s_full[kAsk], s_empty[kAsk], i_full[kInfo], i_empty[kInfo], fin;
    uint32_t tmem_slot;
    int abort_flag;
};

struct Params {
    const int* offsets;
    const int* order;           /* gathered rows (NULL: sorted) */
    int top_k, m, experts;
    const void* x;              /* gathered rows: xcols elements, ldx apart */
    long long ldx;
    int xcols;
    int F, J, C;                /* J: GRADW's rows of one expert's output; C: contraction (not GRADW) */
    void* out;
    long long ldo, stride_o;
    int pairs;                  /* 4-byte stores are aligned */
};

/* Four rows of a 2-D tensor map with a one-row box, 64 elements from x each, to
 * 4 x 128 bytes of shared memory (swizzled by address like any other box). */
__device__ __forceinline__ void tma_gather4_pair(const CUtensorMap* map, uint32_t bar, void* smem, int x,
                                                 const int (&r)[4]) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
        :: "r"(smem_u32(smem)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(r[0]), "r"(r[1]),
           "r"(r[2]), "r"(r[3])
        : "memory");
}
/* 16 bytes of global memory to shared memory, the bytes past `bytes` as zeros (none is read at 0). */
__device__ __forceinline__ void cp_async16(void* smem, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(smem_u32(smem)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
/* Orders this thread's writes to shared memory before later reads by TMA and the tensor cores. */
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tma_load_2d_pair(const CUtensorMap* map, uint32_t bar, void* smem, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];"
        :: "r"(smem_u32(smem)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    int ok = 0;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait(bar, parity, abort_flag, &g_experts_status) ? 1 : 0;
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

/* Arrival on, and wait for, a barrier by which one CTA of a pair tells the other that it may write, or has written,
 * a word of shared memory: release and acquire at the cluster's scope. */
__device__ __forceinline__ void arrive_released(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool wait_acquired(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    if (!mbar_wait(bar, parity, abort_flag, &g_experts_status)) return false;
    uint32_t ok;                                 /* the phase is complete: true at once */
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(bar, parity))
        if (globaltimer() - t0 > kWaitLimitNs) return;
}

/* Asks for the next cluster that has not started; the answer (16 bytes) comes to this
 * CTA's shared memory and counts on its barrier. */
__device__ __forceinline__ void ask_next(uint4* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 :: "r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
/* A word to another CTA of the cluster, counted on its barrier. */
__device__ __forceinline__ void send_word(uint32_t cluster_addr, int v, uint32_t cluster_bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];"
                 :: "r"(cluster_addr), "r"(v), "r"(cluster_bar) : "memory");
}
/* First block of the cluster taken over, or -1: none is left. */
__device__ __forceinline__ int read_next(const uint4* answer) {
    uint32_t yes, x;
    uint4 a;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w) : "r"(smem_u32(answer)) : "memory");
    asm volatile("{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t.reg .b64 lo, hi;\n\t"
                 "mov.b64 lo, {%2, %3};\n\tmov.b64 hi, {%4, %5};\n\tmov.b128 h, {lo, hi};\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
                 : "=r"(yes), "=r"(x) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w));
    return yes ? (int)x : -1;
}
/* The tiles of all experts in the order they are worked on: expert by expert,
 * inside one kGroup row tiles at a time, their f tiles in turn, the row tiles
 * innermost -- clusters that run together then share a few tiles of W and of X, and
 * a weight matrix larger than L2 is read once per kGroup row tiles.  start[e] is
 * the first row tile of expert e, row[e] its first sorted row. */
template <int MODE, int BN, int FTILE>
struct Tiles {
    const int* start;
    const int* row;
    int experts, J, nk;
    int ft;                     /* f tiles */
    int e;
    __device__ Tiles(const Params& p, const int* start_, const int* row_)
        : start(start_), row(row_), experts(p.experts), J(p.J), nk((p.C + BK - 1) / BK), ft((p.F + FTILE - 1) / FTILE), e(0) {}
    /* u mostly ascends from call to call */
    __device__ Tile at(int u) {
        Tile t;
        t.u = u;
        t.e = 0;
        t.r0 = t.rows = t.j0 = t.nj = t.wide = t.f0 = t.nk = 0;
        if (u >= (long long)start[experts] * ft) return t;
        if ((long long)start[e] * ft > u) e = 0;
        while ((long long)start[e + 1] * ft <= u) ++e;
        t.e = e;
        const int l0 = start[e], count = start[e + 1] - l0;
        const int l = (int)(u - (long long)l0 * ft);
        const int g = l / (kGroup * ft);
        const int rem = l - g * kGroup * ft;
        const int in = min(kGroup, count - g * kGroup);
        const int f = rem / in;
        t.f0 = f * FTILE;
        t.j0 = (g * kGroup + rem - f * in) * BN;
        t.r0 = row[e];
        t.rows = max(row[e + 1] - t.r0, 0);
        t.nj = min(BN, (MODE == EXP_GRADW ? J : t.rows) - t.j0);
        t.wide = min(BN, (t.nj + 31) & ~31);
        t.nk = MODE == EXP_GRADW ? (t.rows + BK - 1) / BK : nk;
        return t;
    }
};

/* Waits for a warp's TMEM loads; the registers pass through, so that no use of them
 * can be placed before the wait. */
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {
    static_assert(N == 16 || N == 32, "one load");
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
    if constexpr (N == 32)
        asm volatile("" : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                          "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                          "+r"(r[30]), "+r"(r[31]) :: "memory");
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[N]) {
    if constexpr (N == 32) tmem_ld32(taddr, r);
    else tmem_ld16(taddr, r);
}

__device__ __forceinline__ uint32_t pack2(float a, float b, bool bf16) {
    uint32_t r;
    if (bf16) asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
    else asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
    return r;
}

/* tmB: FWD, GRADX: boxes of 32 rows, tmBg one of 128 for the tiles that need four of
 * those (GRADX of 32768 x 2048 by 4096, 32 experts: 478 us with four, 456 with one).
 * GRADW: tmB 64 x 64 boxes, tmAg and tmBg single rows, tmAt and tmBt the tails. */
template <int MODE, bool PAIR, int BN, int FMT>
__global__ void __launch_bounds__(Cfg<PAIR, BN>::THREADS, 1)
k_experts_tc(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
             const __grid_constant__ CUtensorMap tmAg, const __grid_constant__ CUtensorMap tmBg,
             const __grid_constant__ CUtensorMap tmAt, const __grid_constant__ CUtensorMap tmBt, const Params p) {
    static_assert(PAIR || MODE != EXP_GRADW, "the weights' gradient runs on pairs");
    using K = Cfg<PAIR, BN>;
    constexpr int STAGES = K::STAGES, STAGE = K::STAGE, BL = K::BL;
    constexpr bool A_MN = MODE != EXP_FWD, B_MN = MODE == EXP_GRADW;
    const bool gathers = !PAIR && p.order != nullptr;
    static_assert(sizeof(EMisc<STAGES>) <= 1024, "misc");
    extern __shared__ __align__(1024) uint8_t smem[];
    EMisc<STAGES>& ms = *reinterpret_cast<EMisc<STAGES>*>(smem + STAGES * STAGE);
    int* start = reinterpret_cast<int*>(smem + STAGES * STAGE + 1024);
    int* first = start + MPK_MAX_EXPERTS + 1;
    volatile int* abort_flag = &ms.abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)cluster_rank() : 0;

    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) atomicOr(&g_experts_status, MPK_DEV_TIMEOUT);
        return;
    }
    if (threadIdx.x == 0) {
        /* a stage is full with the TMA bytes and, where rows are gathered, the gather warp's arrival */
        const int arrivals = gathers ? 2 : 1;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&ms.full[i], arrivals); mbar_init(&ms.empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&ms.t_full[i], 1); mbar_init(&ms.t_empty[i], (PAIR ? 2 : 1) * kEpiWarps); }
        /* answers are read by the producers, tiles by this CTA's MMA issuer (in CTA 1 the warp that would be it),
         * epilogue and gather warps */
        for (int i = 0; i < kAsk; ++i) { mbar_init(&ms.s_full[i], 1); mbar_init(&ms.s_empty[i], PAIR ? 2 : 1); }
        const int readers = 1 + kEpiWarps + (gathers ? kGatherWarps : 0);
        for (int i = 0; i < kInfo; ++i) { mbar_init(&ms.i_full[i], 1); mbar_init(&ms.i_empty[i], readers); }
        mbar_init(&ms.fin, 1);
        ms.abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) { tma_prefetch_desc(&tmA); tma_prefetch_desc(&tmB); }
    if (warp == 1) {
        if (PAIR) tmem_alloc_pair(&ms.tmem_slot, K::TMEM_COLS);
        else tmem_alloc(&ms.tmem_slot, K::TMEM_COLS);
    }
    if (warp == 2) {                             /* first row tile and first row of every expert */
        int run = 0;
        for (int e0 = 0; e0 < p.experts; e0 += 32) {
            const int e = e0 + lane;
            int t = 0;
            if (e < p.experts) {
                const int r = expert_start(p.offsets, e, p.m);
                const int rows = MODE == EXP_GRADW ? p.J : max(expert_start(p.offsets, e + 1, p.m) - r, 0);
                t = (rows + BN - 1) / BN;
                first[e] = r;
            }
            int incl = t;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (e < p.experts) start[e] = min(run + incl - t, kMostTiles);
            run = min(run + __shfl_sync(0xffffffffu, incl, 31), kMostTiles);
        }
        if (lane == 0) {
            start[p.experts] = run;
            first[p.experts] = expert_start(p.offsets, p.experts, p.m);
        }
    }
    tc_fence_before();
    if (PAIR) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = ms.tmem_slot;

    /* The next tile, for a whole warp or (LONE) for its lane 0 alone; false when there is none or a wait
     * ran out. */
    int taken = 0;
    auto take = [&](Tile& t, bool lone) {
        const int sl = taken % kInfo;
        const uint32_t parity = (uint32_t)(taken / kInfo) & 1u;
        ++taken;
        if (lone ? !mbar_wait(&ms.i_full[sl], parity, abort_flag, &g_experts_status)
                 : !wait_warp(&ms.i_full[sl], parity, abort_flag)) return false;
        t = ms.info[sl];
        if (!lone) __syncwarp();
        if (lane == 0) mbar_arrive(&ms.i_empty[sl]);
        return t.u >= 0;
    };

    if (warp == 0) {
        /* ------------------------------------------------- producer ---- */
        Tiles<MODE, BN, K::FT> tiles(p, start, first);
        uint32_t last[STAGES];
#pragma unroll
        for (int i = 0; i < STAGES; ++i) last[i] = 0xffffffffu;
        uint32_t it = 0;
        int u = PAIR ? blockIdx.x >> 1 : blockIdx.x;
        int told = 0, asked = 0;                 /* tiles passed on, indices asked for */
        bool ok = true;
        while (ok) {
            /* The next index is asked for as this tile starts, no earlier: once given it is this cluster's. */
            if (lane == 0 && rank == 0 && u >= 0) {
                const int sl = asked % kAsk;
                const uint32_t parity = ((uint32_t)(asked / kAsk) & 1u) ^ 1u;
                ok = PAIR ? wait_acquired(&ms.s_empty[sl], parity, abort_flag)
                          : mbar_wait(&ms.s_empty[sl], parity, abort_flag, &g_experts_status);
                if (ok) {
                    mbar_expect_tx(&ms.s_full[sl], 16);
                    ask_next(&ms.next[sl], &ms.s_full[sl]);
                }
            }
            if (!__shfl_sync(0xffffffffu, ok ? 1 : 0, 0)) { ok = false; break; }
            if (u >= 0) ++asked;
            Tile t = tiles.at(u < 0 ? 0x7fffffff : u);
            t.u = u;
            {
                const int sl = told % kInfo;
                if (!wait_warp(&ms.i_empty[sl], ((uint32_t)(told / kInfo) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                if (lane == 0) {
                    ms.info[sl] = t;
                    mbar_arrive(&ms.i_full[sl]);
                }
                ++told;
            }
            if (u < 0) break;
            const int f0 = t.f0 + rank * BM;                     /* this CTA's f's */
            const int jn = PAIR ? t.wide / 2 : BN;               /* and j's */
            const int jl = t.j0 + rank * jn;
            const int end = t.r0 + t.rows;
            const int boxes = MODE == EXP_GRADW ? (jn + 63) / 64 : (jn + BROWS - 1) / BROWS;
            const uint32_t bytes = A_STAGE + (gathers ? 0 : boxes * (MODE == EXP_GRADW ? BOX : BROWS * BK * 2));
            /* GRADW's last stage: lane l fetches rows 4 (l mod 16) .. of the 64-element chunk l / 16 */
            const int q4 = 4 * (lane & 15), ch = lane >> 4;
            for (int kc = 0; kc < t.nk; ++kc, ++it) {
                const int st = (int)(it % STAGES);
                const uint32_t use = it / STAGES;
                if (!wait_warp(&ms.empty[st], (use & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                uint8_t* sa = smem + st * STAGE;
                uint8_t* sb = sa + A_STAGE;
                uint64_t* bar = &ms.full[st];
                const uint32_t pbar = PAIR ? peer_addr(bar, 0) : 0u;
                if (lane == 0) {
                    if (!PAIR) mbar_expect_tx(bar, bytes);
                    else if (rank == 0) mbar_expect_tx(bar, 2 * bytes);
#pragma unroll
                    for (int i = 0; i < STAGES; ++i)
                        if (i == st) last[i] = use;
                }
                __syncwarp();
                auto load3 = [&](const CUtensorMap* map, void* dst, int x, int y, int z) {
                    if (PAIR) tma_load_3d_pair(map, pbar, dst, x, y, z);
                    else tma_load_3d(map, bar, dst, x, y, z);
                };
                auto load2 = [&](const CUtensorMap* map, void* dst, int x, int y) {
                    if (PAIR) tma_load_2d_pair(map, pbar, dst, x, y);
                    else tma_load_2d(map, bar, dst, x, y);
                };
                if (MODE != EXP_GRADW) {
                    if (lane == 0) {
                        if (MODE == EXP_FWD) {
                            load3(&tmA, sa, kc * BK, f0, t.e);
                        } else {
                            load3(&tmA, sa, f0, kc * BK, t.e);
                            load3(&tmA, sa + BOX, f0 + 64, kc * BK, t.e);
                        }
                    }
                    if (BL == 128 && boxes == 128 / BROWS) {
                        if (lane == 0) load2(&tmBg, sb, kc * BK, t.r0 + jl);
                    } else if (!gathers && lane < boxes) {
                        load2(&tmB, sb + lane * (BROWS * BK * 2), kc * BK, t.r0 + jl + BROWS * lane);
                    }
                } else {
                    const int r = t.r0 + kc * BK;
                    if (r + BK <= end) {
                        if (lane < 2) load2(&tmA, sa + lane * BOX, f0 + 64 * lane, r);
                        if (lane < boxes) load2(&tmB, sb + lane * BOX, jl + 64 * lane, r);
                    } else if (end >= BK) {
                        const int y = BK - (end - r), z = end - BK;
                        if (lane < 2) load3(&tmAt, sa + lane * BOX, f0 + 64 * lane, y, z);
                        if (lane < boxes) load3(&tmBt, sb + lane * BOX, jl + 64 * lane, y, z);
                    } else {
                        int own[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) own[i] = r + q4 + i < end ? r + q4 + i : p.m;
                        tma_gather4_pair(&tmAg, pbar, sa + ch * BOX + q4 * 128, f0 + 64 * ch, own);
                        if (ch < boxes) tma_gather4_pair(&tmBg, pbar, sb + ch * BOX + q4 * 128, jl + 64 * ch, own);
                    }
                }
            }
            if (!ok) break;
            /* the answer to this tile's question */
            const int sl = (asked - 1) % kAsk;
            int x = -1, got = 0;
            if (lane == 0) {
                if (rank == 1) mbar_expect_tx(&ms.s_full[sl], 4);
                const uint32_t parity = (uint32_t)((asked - 1) / kAsk) & 1u;
                if (rank == 1) got = wait_acquired(&ms.s_full[sl], parity, abort_flag) ? 1 : 0;
                else got = mbar_wait(&ms.s_full[sl], parity, abort_flag, &g_experts_status) ? 1 : 0;
                if (got && rank == 1) {
                    x = *const_cast<volatile int*>(&ms.passed[sl]);     /* warp 1 says so to CTA 0 */
                } else if (got) {
                    x = read_next(&ms.next[sl]);
                    fence_async_proxy();
                    if (PAIR) send_word(peer_addr(&ms.passed[sl], 1), x, peer_addr(&ms.s_full[sl], 1));
                    mbar_arrive(&ms.s_empty[sl]);
                }
            }
            ok = __shfl_sync(0xffffffffu, got, 0) != 0;
            x = __shfl_sync(0xffffffffu, x, 0);
            u = x < 0 ? -1 : PAIR ? x >> 1 : x;
        }
        if (!ok && lane == 0) {
            /* let what is in flight land before the CTA exits */
            if (asked > 0 && rank == 0) drain_wait(&ms.s_full[(asked - 1) % kAsk], (uint32_t)((asked - 1) / kAsk) & 1u);
            if (!PAIR) {
#pragma unroll
                for (int i = 0; i < STAGES; ++i)
                    if (last[i] != 0xffffffffu) drain_wait(&ms.full[i], last[i] & 1u);
            } else {
                /* a pair's loads complete on CTA 0's barriers, and a phase that was never armed does not
                 * complete: give every load in flight a fixed time (each takes microseconds) */
                const unsigned long long t_end = globaltimer() + 20000000ull;
                while (globaltimer() < t_end) {
                }
            }
        }
    } else if (warp == 1) {
        /* ------------------------------------------------- MMA issuer --- */
        if (lane == 0 && rank == 0) {
            auto commit = [&](uint64_t* bar) {
                if (PAIR) {
                    umma_commit_pair(peer_addr(bar, 0));
                    umma_commit_pair(peer_addr(bar, 1));
                } else {
                    umma_commit(bar);
                }
            };
            uint32_t it = 0, ts = 0;
            bool ok = true;
            Tile t;
            while (ok && take(t, true)) {
                if (t.nk == 0 || t.nj == 0) continue;
                const int tb = (int)(ts & 1u);
                if (!mbar_wait(&ms.t_empty[tb], ((ts >> 1) & 1u) ^ 1u, abort_flag, &g_experts_status)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (uint32_t)(tb * BN);
                const uint32_t idesc = idesc_f16(PAIR ? 2 * BM : BM, t.wide, FMT, A_MN ? 1 : 0, B_MN ? 1 : 0);
                for (int kc = 0; kc < t.nk; ++kc, ++it) {
                    const int st = (int)(it % STAGES);
                    if (!mbar_wait(&ms.full[st], (it / STAGES) & 1u, abort_flag, &g_experts_status)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + st * STAGE);
                    const uint32_t sb = sa + A_STAGE;
#pragma unroll
                    for (int ks = 0; ks < BK / 16; ++ks) {
                        const uint64_t ad = A_MN ? sw128_desc(sa + ks * 2048, BOX, 1024) : sw128_desc(sa + ks * 32, 16, 1024);
                        const uint64_t bd = B_MN ? sw128_desc(sb + ks * 2048, BOX, 1024) : sw128_desc(sb + ks * 32, 16, 1024);
                        const uint32_t acc = (kc > 0 || ks > 0) ? 1u : 0u;
                        if (PAIR) umma_f16_pair(d_tmem, ad, bd, idesc, acc);
                        else umma_f16(d_tmem, ad, bd, idesc, acc);
                    }
                    commit(&ms.empty[st]);
                }
                if (ok) commit(&ms.t_full[tb]);
                ++ts;
            }
            if (PAIR) umma_commit_pair(peer_addr(&ms.fin, 0));
            else umma_commit(&ms.fin);
            drain_wait(&ms.fin, 0);
        }
        if (PAIR && lane == 0 && rank == 1) {
            /* CTA 1's MMA issuer has no MMAs: it tells CTA 0 that a passed index was read, once the producer has
             * passed on that tile.  (The release at the cluster's scope waits for the SM's stores: in the producer
             * it cost the gradient of 64 x 1024 x 2048 weights 4 %.) */
            for (int n = 0;; ++n) {
                const int sl = n % kInfo;
                if (!mbar_wait(&ms.i_full[sl], (uint32_t)(n / kInfo) & 1u, abort_flag, &g_experts_status)) break;
                const int u = ms.info[sl].u;
                mbar_arrive(&ms.i_empty[sl]);
                if (n > 0) arrive_released(peer_addr(&ms.s_empty[(n - 1) % kAsk], 0));
                if (u < 0) break;
            }
        }
    } else if (warp >= 2 + kEpiWarps) {
        /* ----------------------------------------------------- gather --- */
        /* Warp w copies the stages of its ring slots on its own.  Lane l copies the 16-byte piece c = l mod
         * 8 of rows l / 8, l / 8 + 4, ...: eight pieces make the 128 bytes a row has in a stage, at place c ^
         * (row mod 8) of them. */
        if constexpr (MODE == EXP_FWD && !PAIR) if (gathers) {
            constexpr int N = BL / 4;                            /* rows a lane */
            static_assert(BL == 32, "a lane looks one row up");
            const int w = warp - (2 + kEpiWarps);
            static_assert(STAGES >= kGatherWarps, "every gather warp has a slot");
            /* the next stage in one of this warp's slots */
            auto after = [&](uint32_t it) {
                const int st = (int)(it % STAGES);
                return it + (uint32_t)(st + kGatherWarps < STAGES ? kGatherWarps : STAGES - st + w);
            };
            const int c = lane & 7, row = lane >> 3;
            const uint16_t* x = static_cast<const uint16_t*>(p.x);
            uint32_t it0 = 0, it = (uint32_t)w;                  /* first stage of the tile; this warp's next */
            bool ok = true;
            int idx[N];
            Tile t;
            while (ok && take(t, false)) {
                const int end = t.r0 + t.rows;
                const uint32_t it1 = it0 + (uint32_t)t.nk;
                if (it < it1) {                                  /* token rows, -1 past the segment */
                    const int at = t.r0 + t.j0 + lane;
                    const int entry = at < end ? p.order[at] : -1;
                    const int own = (unsigned)entry < (unsigned)p.m ? entry / p.top_k : -1;
#pragma unroll
                    for (int i = 0; i < N; ++i) idx[i] = __shfl_sync(0xffffffffu, own, 4 * i + row);
                }
                for (; it < it1; it = after(it)) {
                    const int kc = (int)(it - it0);
                    const int st = (int)(it % STAGES);
                    if (!wait_warp(&ms.empty[st], ((it / STAGES) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                    uint8_t* dst = smem + st * STAGE + A_STAGE;
                    const int col = kc * BK + 8 * c;
                    const int bytes = min(16, max(0, 2 * (p.xcols - col)));
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int r = row + 4 * i;
                        const bool there = idx[i] >= 0 && bytes > 0;
                        cp_async16(dst + r * 128 + ((c ^ (r & 7)) << 4),
                                   there ? x + (long long)idx[i] * p.ldx + col : x, there ? bytes : 0);
                    }
                    cp_async_wait_all();
                    fence_async_proxy();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ms.full[st]);
                }
                it0 = it1;
            }
            cp_async_wait_all();
        }
    } else {
        /* --------------------------------------------------- epilogue --- */
        constexpr int CH = K::CH, HALF = K::HALF;
        const int half = (warp - 2) >> 2;         /* which columns of the tile */
        const int q = warp & 3;                   /* TMEM lane quarter */
        const uint32_t t_lane = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * HALF);
        const int odd = lane & 1;
        const uint32_t sel = odd ? 0x3276u : 0x5410u;
        const int units = PAIR ? gridDim.x >> 1 : gridDim.x;
        const int valid = first[p.experts];
        const long long two = 2 * p.ldo;
        uint16_t* out = static_cast<uint16_t*>(p.out);
        bool ok = true;
        uint32_t ts = 0;
        Tile t;
        while (ok && take(t, false)) {
            if (MODE != EXP_GRADW) {              /* rows that no expert owns: each index sets its share to zero */
                for (long long r = (long long)valid + t.u; r < p.m; r += units)
                    for (int f = rank * 32 * kEpiWarps + (int)threadIdx.x - 64; f < p.F; f += (PAIR ? 2 : 1) * 32 * kEpiWarps)
                        out[r * p.ldo + f] = 0;
            }
            if (t.nj == 0) continue;
            const int f = t.f0 + rank * BM + q * 32 + lane;
            uint16_t* base = MODE == EXP_GRADW ? out + (long long)t.e * p.stride_o + (long long)t.j0 * p.ldo
                                               : out + (long long)(t.r0 + t.j0) * p.ldo;
            const int nj = t.nj - half * HALF;                   /* columns of this warp that exist */
            base += (long long)(half * HALF) * p.ldo;
            /* the whole warp's 32 f's exist */
            const bool inside = p.pairs && t.f0 + rank * BM + q * 32 + 32 <= p.F;
            auto put = [&](const uint32_t (&r)[CH], int c) {
                if (p.pairs) {
                    /* columns e, e + 1 of this lane's f and of its neighbour's: the even lane takes column e
                     * of both, the odd lane column e + 1 */
                    uint32_t v[CH / 2];
#pragma unroll
                    for (int e = 0; e < CH; e += 2) {
                        const uint32_t own = pack2(__uint_as_float(r[e]), __uint_as_float(r[e + 1]), FMT == 1);
                        v[e / 2] = __byte_perm(own, __shfl_xor_sync(0xffffffffu, own, 1), sel);
                    }
                    const int fe = f - odd;
                    uint16_t* dst = base + (long long)(c + odd) * p.ldo + fe;
                    if (inside && c + CH <= nj) {
#pragma unroll
                        for (int e = 0; e < CH / 2; ++e, dst += two) *reinterpret_cast<uint32_t*>(dst) = v[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < CH / 2; ++e, dst += two)
                            if (c + 2 * e + odd < nj) {
                                if (fe + 1 < p.F) *reinterpret_cast<uint32_t*>(dst) = v[e];
                                else if (fe < p.F) *dst = (uint16_t)v[e];
                            }
                    }
                } else {
                    uint16_t* dst = base + (long long)c * p.ldo + f;
#pragma unroll
                    for (int e = 0; e < CH; ++e) {
                        if (c + e < nj && f < p.F) *dst = (uint16_t)pack2(__uint_as_float(r[e]), 0.f, FMT == 1);
                        dst += p.ldo;
                    }
                }
            };
            if (t.nk == 0) {                                     /* an expert without rows */
                uint32_t r[CH];
#pragma unroll
                for (int e = 0; e < CH; ++e) r[e] = 0u;
#pragma unroll 1
                for (int c = 0; c < HALF && c < nj; c += CH) put(r, c);
                continue;
            }
            const int tb = (int)(ts & 1u);
            if (!wait_warp(&ms.t_full[tb], (ts >> 1) & 1u, abort_flag)) { ok = false; break; }
            ++ts;
            tc_fence_after();
            /* the accumulator is free again once its last columns are in registers */
            auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_cluster(peer_addr(&ms.t_empty[tb], 0));
                    else mbar_arrive(&ms.t_empty[tb]);
                }
            };
            const uint32_t col = t_lane + (uint32_t)(tb * BN);
            if (nj <= 0) {
                release();
                continue;
            }
            const int chunks = min(HALF / CH, (nj + CH - 1) / CH);
            uint32_t r[2][CH];
            tmem_load(col, r[0]);
#pragma unroll
            for (int c = 0; c < HALF / CH; ++c) {
                if (c < chunks) {
                    tmem_wait(r[c & 1]);
                    if (c + 1 < chunks) tmem_load(col + (uint32_t)((c + 1) * CH), r[(c + 1) & 1]);
                    else release();
                    put(r[c & 1], c * CH);
                }
            }
        }
    }

    tc_fence_before();
    if (PAIR) cluster_sync();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        if (PAIR) tmem_dealloc_pair(tmem_base, K::TMEM_COLS);
        else tmem_dealloc(tmem_base, K::TMEM_COLS);
    }
}

/* ------------------------------------------------------------- host side ---- */

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* q = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &q, 12000, cudaEnableDefault, &res) == cudaSuccess &&
            res == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(q);
    });
    return fn;
}

/* rows x cols (x planes) with row stride ld and plane stride, 64-element boxes of box_rows rows. */
bool row_map(CUtensorMap* map, const void* base, bool bf16, long long cols, long long rows, long long planes, long long ld,
             long long stride, int box_rows) {
    auto fn = encode_fn();
    if (!fn) return false;
    if (rows <= 1) ld = (cols + 7) / 8 * 8;
    if (planes <= 1) stride = ld;                /* no step is ever taken along it */
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    const cuuint32_t es[3] = {1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, planes ? 3 : 2,
              const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE, bool PAIR, int BN, int FMT>
cudaError_t launch_t(const ExpertArgs& a, cudaStream_t s) {
    using K = Cfg<PAIR, BN>;
    auto kern = k_experts_tc<MODE, PAIR, BN, FMT>;
    CUtensorMap tmA{}, tmB{}, tmAg{}, tmBg{}, tmAt{}, tmBt{};
    bool ok;
    if (MODE == EXP_FWD) {
        ok = row_map(&tmA, a.w, a.bf16, a.k, a.width, a.experts, a.ldw, a.stride_w, BM) &&
             (a.order || (row_map(&tmB, a.x, a.bf16, a.k, a.m, 0, a.ldx, 0, BROWS) &&
                          row_map(&tmBg, a.x, a.bf16, a.k, a.m, 0, a.ldx, 0, 128)));
    } else if (MODE == EXP_GRADX) {
        ok = row_map(&tmA, a.w, a.bf16, a.k, a.width, a.experts, a.ldw, a.stride_w, BK) &&
             row_map(&tmB, a.gy, a.bf16, a.width, a.m, 0, a.ldgy, 0, BROWS) &&
             row_map(&tmBg, a.gy, a.bf16, a.width, a.m, 0, a.ldgy, 0, 128);
    } else {
        ok = row_map(&tmA, a.x, a.bf16, a.k, a.m, 0, a.ldx, 0, BK) && row_map(&tmAg, a.x, a.bf16, a.k, a.m, 0, a.ldx, 0, 1) &&
             row_map(&tmB, a.gy, a.bf16, a.width, a.m, 0, a.ldgy, 0, BK) &&
             row_map(&tmBg, a.gy, a.bf16, a.width, a.m, 0, a.ldgy, 0, 1);
        if (a.m >= BK)                           /* rows y + z, y < 64, z <= m - 64: all inside the matrix */
            ok = ok && row_map(&tmAt, a.x, a.bf16, a.k, BK, a.m - BK + 1, a.ldx, a.ldx, BK) &&
                 row_map(&tmBt, a.gy, a.bf16, a.width, BK, a.m - BK + 1, a.ldgy, a.ldgy, BK);
    }
    if (!ok) return cudaErrorInvalidValue;
    Params p{a.offsets, a.order, a.top_k, (int)a.m, a.experts, a.x, a.ldx, a.k, MODE == EXP_FWD ? a.width : a.k, a.width,
             MODE == EXP_FWD ? a.k : a.width, a.out, a.ldo, a.stride_o,
             reinterpret_cast<uintptr_t>(a.out) % 4 == 0 && a.ldo % 2 == 0 && (MODE != EXP_GRADW || a.stride_o % 2 == 0)};
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, K::SMEM_BYTES);
    if (e != cudaSuccess) return e;
    /* a cluster for every tile there can be: every expert with rows rounds up by one */
    const long long ft = (p.F + K::FT - 1) / K::FT;
    const long long some = a.m < a.experts ? a.m : a.experts;
    const long long jt = MODE == EXP_GRADW ? (long long)a.experts * ((a.width + BN - 1) / BN) : a.m / BN + some;
    const long long units = ft * jt;
    if (units > (1LL << 30)) return cudaErrorInvalidConfiguration;
    const int n = (int)units;
    if (!PAIR) {
        kern<<<n, K::THREADS, K::SMEM_BYTES, s>>>(tmA, tmB, tmAg, tmBg, tmAt, tmBt, p);
        return cudaGetLastError();
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(2 * n, 1, 1);
    cfg.blockDim = dim3(K::THREADS, 1, 1);
    cfg.dynamicSmemBytes = K::SMEM_BYTES;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmAg, tmBg, tmAt, tmBt, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

/* Tile widths by the average expert's rows.  A pair's 64-wide tile has ten stages of
 * W in flight, the 256-wide one six.  Measured, 64 experts of 1024 x 2048, GRADX:
 * 1 row an expert 39 us on 32-wide tiles and 38 on 256-wide pairs, 6 rows 63, 57 and
 * 52 on 64-wide pairs, 20 rows 76, 58 and 58, 64 rows 70 on 64-wide and 61 on
 * 256-wide pairs.  FWD gathers rows itself on 32-wide tiles, which the copy of a
 * sorted X must be weighed against: 12 rows 60 us there, 67 on pairs with the copy,
 * 16 rows 72 and 64. */
template <int FMT>
cudaError_t launch_fmt(const ExpertArgs& a, cudaStream_t s) {
    const long long rows = a.m / a.experts;
    if (a.mode == EXP_GRADW) return launch_t<EXP_GRADW, true, 256, FMT>(a, s);
    if (a.mode == EXP_GRADX) {
        if (rows <= 2) return launch_t<EXP_GRADX, false, 32, FMT>(a, s);
        return rows <= 48 ? launch_t<EXP_GRADX, true, 64, FMT>(a, s) : launch_t<EXP_GRADX, true, 256, FMT>(a, s);
    }
    if (experts_few_rows(a.m, a.experts)) return launch_t<EXP_FWD, false, 32, FMT>(a, s);
    return rows <= 48 ? launch_t<EXP_FWD, true, 64, FMT>(a, s) : launch_t<EXP_FWD, true, 256, FMT>(a, s);
}

bool rows16(const void* q, long long ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 8 == 0; }

}  /* namespace */

bool experts_few_rows(long long m, int experts) { return m / experts <= 12; }

bool experts_tc_ok(const ExpertArgs& a) {
    /* TMA addresses and strides: 16-byte steps, strides below 2^40 bytes; one row has no stride */
    const long long most = 1LL << 38;
    const long long xrows = a.order ? a.m / a.top_k : a.m;
    const bool x = a.mode == EXP_GRADX || rows16(a.x, xrows > 1 ? a.ldx : 8);
    const bool gy = a.mode == EXP_FWD || rows16(a.gy, a.m > 1 ? a.ldgy : 8);
    const bool w = a.mode == EXP_GRADW ||
                   (rows16(a.w, a.width > 1 ? a.ldw : 8) && (a.experts == 1 || a.stride_w % 8 == 0));
    return x && gy && w && a.ldx < most && a.ldgy < most && a.ldw < most && a.stride_w < most && a.m > 0;
}

cudaError_t launch_experts_tc(const ExpertArgs& a, cudaStream_t s) {
    return a.bf16 ? launch_fmt<1>(a, s) : launch_fmt<0>(a, s);
}

}  /* namespace mpk */

extern "C" int mpkDebugExpertStatus(int clear) {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, mpk::g_experts_status, sizeof(int)) != cudaSuccess) return -1;
    if (clear) {
        const int zero = 0;
        if (cudaMemcpyToSymbol(mpk::g_experts_status, &zero, sizeof(int)) != cudaSuccess) return -1;
    }
    return v;
}
