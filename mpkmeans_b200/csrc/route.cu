/* route.cu -- tokens routed to experts: choice and weights, their gradient, and
 * the plan that sorts the routed rows by expert (include/mpkexperts.h).
 *
 * mpkRoute, one warp a token.  With logits l, scores s (softmax or sigmoid) and
 * choice values c = s + bias, the warp keeps the row in registers (experts VPL *
 * lane ... in registers 0 ..), turns every choice value into an integer key of the same
 * order (NaN highest, masked lowest) and drops the groups that lose.  The top_k
 * largest of the 32 lanes' maxima give a bound that at least top_k experts reach
 * and few others do: about ten of 256 for top_k = 8.  Those are packed one a lane
 * and ranked against each other.  (Taking the maximum top_k times, rescanning the
 * registers of the lane that held it, was a third of 1800 instructions a row.)
 * Bound by instruction issue: 32768 x 256 FP32 takes 24 us with softmax, 41 to 47 with
 * sigmoid, bias and groups.  Equal biases with BF16 logits, whose ties send many rows
 * to slow_choice, 37 to 39 us without groups and up to 66 with; 1024 experts with a
 * bias 184 to 242 us.
 *
 * The choice is exact, as the assignment's is: without a bias, and with groups
 * scored by their maximum, the order of c is the order of l and the keys are the
 * logits themselves.  Otherwise c is an FP32 evaluation with a bounded error; a
 * row in which two neighbours of the chosen sequence (the first loser included)
 * or the groups on both sides of the cut come within twice that bound is
 * decided again in FP64 (slow_choice), except where the two have the same logit
 * and the same bias, which is an exact tie.  A tie of the last slot with the
 * first loser says nothing of the losers behind: those within the bound of the
 * tie that the logits' order does not settle send the row to FP64 too, and so
 * does any other near pair of it.  The scores of a 256-expert row lie some 1e-3
 * apart and the bound is about 1e-6, so few rows go there.
 */
#include "experts.cuh"
#include "mpkexperts.h"

#include <climits>
#include <cmath>
#include <type_traits>

namespace mpk {
namespace {

constexpr unsigned FULL = 0xffffffffu;
constexpr int kRouteWarps = 4;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

/* An unsigned key in the order of v: the two zeros equal, NaN the highest (the
 * addition makes every NaN the positive one), -inf below kLive. */
constexpr unsigned kLive = 0x00800000u;
__device__ __forceinline__ unsigned key_of(float v) {
    const unsigned u = __float_as_uint(v + 0.0f);
    return u ^ (0x80000000u | (unsigned)((int)u >> 31));
}
__device__ __forceinline__ float of_key(unsigned k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
/* The same in FP64, -inf as 0. */
__device__ __forceinline__ unsigned long long key_of(double v) {
    if (v != v) return ~0ull;
    const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
    const unsigned long long k = (u >> 63) ? ~u : (u | (1ull << 63));
    return v == -(double)INFINITY ? 0ull : k;
}
__device__ __forceinline__ double of_key(unsigned long long k) {
    if (k == ~0ull) return (double)NAN;
    if (k == 0ull) return -(double)INFINITY;
    return __longlong_as_double((long long)((k >> 63) ? (k & ~(1ull << 63)) : ~k));
}

__device__ __forceinline__ bool live(unsigned k) { return k >= kLive; }
__device__ __forceinline__ bool live(unsigned long long k) { return k != 0; }

__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

struct RouteShape {
    int E, k, score, G, gs, top_groups, group_score, renorm;
    unsigned gmul;            /* group of expert j: (j * gmul) >> 20, exact for j, gs < 1024 */
    float scale;
    int log_l;                /* lanes a group scan takes (log2): 2^log_l * G <= 32 */
    int log_k;                /* lanes the slots take (log2): 2^log_k >= k */
    int log_g;                /* lanes that hold one group, where whole lanes do and their number is a power
                               * of two (log2); -1: groups go through shared memory */
    int vec;                  /* a lane's experts can be loaded and stored as one word or as 16-byte words */
};

/* Sum, maximum over the slots' lanes (the others hold the neutral value). */
__device__ __forceinline__ float slot_sum(float v, int log_k) {
    for (int o = (1 << log_k) >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
__device__ __forceinline__ float slot_max(float v, int log_k) {
    for (int o = (1 << log_k) >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
    return v;
}

/* A lane's VPL consecutive elements of a row, from element VPL * lane. */
template <typename T, int VPL>
struct LaneRow {
    static constexpr int BYTES = VPL * (int)sizeof(T);
    static constexpr int WORD = BYTES < 16 ? BYTES : 16;
    using W = typename std::conditional<WORD == 2, unsigned short, typename std::conditional<WORD == 4, unsigned,
              typename std::conditional<WORD == 8, uint2, uint4>::type>::type>::type;
    /* -inf past the row */
    __device__ static __forceinline__ void load(const T* row, int E, bool vec, int lane, float (&x)[VPL]) {
        const int j = VPL * lane;
        if (vec && j + VPL <= E) {
            W w[BYTES / WORD];
#pragma unroll
            for (int i = 0; i < BYTES / WORD; ++i) w[i] = reinterpret_cast<const W*>(row + j)[i];
            const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
            for (int v = 0; v < VPL; ++v) x[v] = to_f(t[v]);
        } else {
#pragma unroll
            for (int v = 0; v < VPL; ++v) x[v] = j + v < E ? to_f(row[j + v]) : -INFINITY;
        }
    }
    __device__ static __forceinline__ void store(T* row, int E, bool vec, int lane, const float (&x)[VPL]) {
        const int j = VPL * lane;
        if (vec && j + VPL <= E) {
            W w[BYTES / WORD];
            T* t = reinterpret_cast<T*>(w);
#pragma unroll
            for (int v = 0; v < VPL; ++v) t[v] = from_f<T>(x[v]);
#pragma unroll
            for (int i = 0; i < BYTES / WORD; ++i) reinterpret_cast<W*>(row + j)[i] = w[i];
        } else {
#pragma unroll
            for (int v = 0; v < VPL; ++v)
                if (j + v < E) row[j + v] = from_f<T>(x[v]);
        }
    }
};

/* The two largest of two pairs (a >= b). */
template <typename KEY>
__device__ __forceinline__ void merge2(KEY& a, KEY& b, KEY a2, KEY b2) {
    if (a2 > a) { b = a > b2 ? a : b2; a = a2; }
    else b = a2 > b ? a2 : b;
}
/* Key of a group from those of its two best. */
template <typename KEY>
__device__ __forceinline__ KEY group_of_two(KEY a, KEY b, int group_score) {
    return group_score == MPK_GROUP_TOP2 && live(b) ? key_of(of_key(a) + of_key(b)) : a;
}

/* The groups' keys (key of the maximum, or of the sum of the two best) from the
 * experts' keys in shared memory: 2^log_l lanes work on a group and all return its
 * key; lanes past the groups return 0.  KEY is the 32-bit key of a float or the
 * 64-bit key of a double. */
template <typename KEY>
__device__ __forceinline__ KEY group_key(const KEY* keys, const RouteShape& sh, int lane) {
    const int L = 1 << sh.log_l, g = lane >> sh.log_l, sub = lane & (L - 1);
    KEY a = 0, b = 0;
    if (g < sh.G)
        for (int i = sub; i < sh.gs; i += L) {
            const KEY v = keys[g * sh.gs + i];
            if (v > a) { b = a; a = v; }
            else if (v > b) b = v;
        }
    for (int o = L >> 1; o > 0; o >>= 1) {
        const KEY a2 = __shfl_xor_sync(FULL, a, o), b2 = __shfl_xor_sync(FULL, b, o);
        merge2(a, b, a2, b2);
    }
    return group_of_two(a, b, sh.group_score);
}

/* Whether this lane's group, lane >> log, is among the top_groups best of G (ties to
 * the lowest index) and has an expert left: the best is taken top_groups times. */
__device__ __forceinline__ bool group_kept(unsigned gk, const RouteShape& sh, int log, int lane) {
    unsigned left = (lane >> log) < sh.G ? gk : 0u;
    bool in = false;
    auto best = [&]() {
        const unsigned m = __reduce_max_sync(FULL, left);
        const int l = __ffs(__ballot_sync(FULL, left == m)) - 1;
        if (live(m) && (lane ^ l) >> log == 0) { in = true; left = 0u; }
    };
    /* the first ones without a loop: branches that the compiler cannot see to be uniform cost a warp
     * synchronisation at every warp-wide operation behind them */
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < sh.top_groups) best();
    for (int i = 4; i < sh.top_groups; ++i) best();
    return in;
}
__device__ __forceinline__ bool group_kept(unsigned long long gk, const RouteShape& sh, int log, int lane) {
    const int g = lane >> log;
    int rank = 0;
    for (int h = 0; h < sh.G; ++h) {
        const unsigned long long o = __shfl_sync(FULL, gk, h << log);
        rank += (o > gk || (o == gk && h < g)) ? 1 : 0;
    }
    return g < sh.G && live(gk) && rank < sh.top_groups;
}

/* The choice of one row in FP64: slot `lane`'s expert, or -1.  keys: E 64-bit words
 * of this warp's shared memory.  Slot `lane` has `mine` so far, slot k being the
 * first loser, and `close` says that the next slot's value is close; where that is
 * no exact tie (the same logit and bias) the order is decided again, and so is the
 * whole choice where the first loser is involved, as the tie of the last slot or in
 * the near pair, or `whole` is set.  (With 32 slots no lane holds the first loser
 * and every row with a bias is decided here.) */
template <typename T>
__device__ __noinline__ int slow_choice(const T* __restrict__ row, const float* __restrict__ bias, RouteShape sh,
                                        unsigned long long* keys, int lane, int mine, bool close, bool whole) {
    const int nj = __shfl_down_sync(FULL, mine, 1);
    const bool tie = close && mine >= 0 && nj >= 0 && to_f(row[mine]) == to_f(row[nj]) && bias[mine] == bias[nj];
    close = close && !tie;
    const bool cut_tie = __any_sync(FULL, tie && lane == sh.k - 1), others = __any_sync(FULL, close);
    whole = whole || (cut_tie && others);
    const bool order_only = !__any_sync(FULL, whole || (close && lane == sh.k - 1));
    if (!__any_sync(FULL, whole || close)) return mine;
    if (lane >= sh.k) mine = -1;
    double mx = 0.0, sum = 1.0;
    if (sh.score == MPK_SCORE_SOFTMAX) {
        float m = -INFINITY;
        for (int j = lane; j < sh.E; j += 32) m = fmaxf(m, to_f(row[j]));
        m = warp_max(m);
        mx = m == -INFINITY ? 0.0 : (double)m;
        sum = 0.0;
        for (int j = lane; j < sh.E; j += 32) sum += exp((double)to_f(row[j]) - mx);
        sum = warp_sum(sum);
    }
    auto key = [&](int j) {
        const double x = (double)to_f(row[j]);
        const double s = sh.score == MPK_SCORE_SOFTMAX ? exp(x - mx) / sum : 1.0 / (1.0 + exp(-x));
        const double c = bias ? s + (double)bias[j] : s;
        return x == -(double)INFINITY ? 0ull : key_of(c);
    };
    if (order_only) {
        const unsigned long long k = mine >= 0 ? key(mine) : 0ull;
        int rank = 0;
        for (int i = 0; i < sh.k; ++i) {
            const unsigned long long k2 = __shfl_sync(FULL, k, i);
            const int j2 = __shfl_sync(FULL, mine, i);
            rank += k2 > k || (k2 == k && j2 < mine) ? 1 : 0;
        }
        if (lane < sh.k && mine >= 0) keys[rank] = (unsigned long long)mine;
        __syncwarp();
        if (mine >= 0 && lane < sh.k) mine = (int)keys[lane];
        __syncwarp();
        return mine;
    }
    for (int j = lane; j < sh.E; j += 32) keys[j] = key(j);
    __syncwarp();
    if (sh.G > 1) {
        const unsigned kept = __ballot_sync(FULL, group_kept(group_key(keys, sh, lane), sh, sh.log_l, lane));
        __syncwarp();
        for (int j = lane; j < sh.E; j += 32) {
            if (!((kept >> (((unsigned)j * sh.gmul >> 20) << sh.log_l)) & 1u)) keys[j] = 0ull;
            else if (!bias) keys[j] = key_of((double)to_f(row[j]));      /* groups chosen: the logits' order again */
        }
        __syncwarp();
    }
    mine = -1;
    for (int i = 0; i < sh.k; ++i) {
        unsigned long long b = 0ull;
        int bj = INT_MAX;
        for (int j = lane; j < sh.E; j += 32)
            if (keys[j] > b) { b = keys[j]; bj = j; }
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long b2 = __shfl_xor_sync(FULL, b, o);
            const int j2 = __shfl_xor_sync(FULL, bj, o);
            if (b2 > b || (b2 == b && j2 < bj)) { b = b2; bj = j2; }
        }
        if (b == 0ull) break;
        if (lane == i) mine = bj;
        if (lane == (bj & 31)) keys[bj] = 0ull;
        __syncwarp();
    }
    __syncwarp();
    return mine;
}

/* 2^x and 1 / x in one instruction each, within 2^-22 and 2^-23 of the value. */
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.44269504f;

/* A chosen score up to a factor that the row's slots share, m being the largest
 * chosen logit: e^(x - m) for softmax, and e^(x - m) / (1 + e^x) for sigmoids that
 * are all below 1/2, whose ratios FP32 then holds wherever their own values would
 * underflow.  As in FP64, a sigmoid below -745 is 0. */
__device__ __forceinline__ float chosen_score(float x, float m, bool softmax) {
    if (softmax) return expf(x - m);
    if (m < 0.f) return x < -745.f ? 0.f : __fdividef(expf(x - m), 1.f + expf(x));
    return __fdividef(1.f, 1.f + expf(-x));
}

/* The `takes` largest of a warp's keys in descending order, the lowest index first
 * among equals: lane i returns the i-th in (key, index), index -1 where there are
 * fewer.  cand: 32 words of this warp's shared memory. */
template <int VPL>
__device__ __forceinline__ void top_keys(unsigned (&key)[VPL], int takes, uint2* cand, int lane, unsigned& mykey,
                                         int& mine) {
    mykey = 0u;
    mine = -1;
    /* bound: the takes-th largest value of the lanes' maxima, or any live key */
    unsigned lm = key[0], bound = kLive;
#pragma unroll
    for (int v = 1; v < VPL; ++v) lm = max(lm, key[v]);
    auto lower = [&]() {
        bound = __reduce_max_sync(FULL, lm);
        if (lm == bound) lm = 0u;
    };
#pragma unroll
    for (int i = 0; i < 9; ++i)
        if (i < takes) lower();
    for (int i = 9; i < takes; ++i) lower();
    bound = max(bound, kLive);
    int own = 0;
#pragma unroll
    for (int v = 0; v < VPL; ++v) own += key[v] >= bound ? 1 : 0;
    int at = own;                                    /* candidates of this and lower lanes */
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(FULL, at, o);
        if (lane >= o) at += u;
    }
    const int count = __shfl_sync(FULL, at, 31);
    at -= own;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        const bool in = key[v] >= bound;
        if (in && at < 32) cand[at] = make_uint2(key[v], (unsigned)(VPL * lane + v));
        at += in ? 1 : 0;
    }
    __syncwarp();
    {
        /* candidate `lane`, in ascending order of index; its rank among them */
        const uint2 c = lane < count ? cand[lane] : make_uint2(0u, 0u);
        int rank = 0;
        auto against = [&](int q) {
            const unsigned o = __shfl_sync(FULL, c.x, q);
            rank += o > c.x || (o == c.x && q < lane) ? 1 : 0;
        };
#pragma unroll
        for (int q = 0; q < 12; ++q) against(q);
        if (count > 12)
            for (int q = 12; q < 32; ++q) against(q);
        __syncwarp();
        if (lane < count && rank < takes) cand[rank] = c;
        __syncwarp();
        if (lane < min(count, takes)) {
            const uint2 m = cand[lane];
            mykey = m.x;
            mine = (int)m.y;
        }
        __syncwarp();
    }
    if (count > 32) {
        /* many equal maxima: the maximum, takes times */
        mykey = 0u;
        mine = -1;
        for (int i = 0; i < takes; ++i) {
            unsigned bk = 0u;
            int bj = INT_MAX;
#pragma unroll
            for (int v = 0; v < VPL; ++v)
                if (key[v] > bk) { bk = key[v]; bj = VPL * lane + v; }
            const unsigned top = __reduce_max_sync(FULL, bk);
            if (top < kLive) break;
            const int j = __reduce_min_sync(FULL, bk == top ? bj : INT_MAX);
            if (lane == i) { mykey = top; mine = j; }
#pragma unroll
            for (int v = 0; v < VPL; ++v)
                if (VPL * lane + v == j) key[v] = 0u;
        }
    }
}

/* Blocks an SM that the registers are cut to, so that slow_choice, which is called
 * from the main path but rarely runs, does not set their number.  (256 experts with
 * a bias: 6, 8, 10 and 12 blocks took 40, 44, 41 and 46 us; without: no difference.
 * Other widths were not tried with other numbers.) */
constexpr int route_blocks(int vpl, bool by_score) { return vpl <= 4 ? 12 : vpl > 8 ? 1 : by_score ? 6 : 10; }

/* BY_SCORE: keys are choice values c (a bias, or groups by their two best), else
 * logits.  GROUPS: 0 none are cut; 1 whole lanes hold a group (log_g >= 0); 2 any
 * others, through shared memory. */
template <typename T, int VPL, bool BY_SCORE, int GROUPS>
__global__ void __launch_bounds__(32 * kRouteWarps, route_blocks(VPL, BY_SCORE))
k_route(const T* __restrict__ logits, long long n, long long ld, const float* __restrict__ bias, RouteShape sh,
        int* __restrict__ ids, float* __restrict__ weights) {
    extern __shared__ unsigned long long route_sm[];
    __shared__ uint2 route_cand[kRouteWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long* keys64 = route_sm + (size_t)warp * sh.E;
    unsigned* keys32 = reinterpret_cast<unsigned*>(keys64);
    const bool softmax = sh.score == MPK_SCORE_SOFTMAX;
    const bool scores = BY_SCORE || (softmax && !sh.renorm);   /* some use of all experts' scores */
    const bool by_logit_after = BY_SCORE && !bias;             /* once groups are chosen, the logits' order again */
    /* the bias of this lane's experts, kept over the rows where registers allow */
    constexpr bool KEEP = BY_SCORE && VPL <= 8;
    float bv[KEEP ? VPL : 1];
    auto bias_of = [&](int v) { return bias && VPL * lane + v < sh.E ? bias[VPL * lane + v] : 0.f; };
    if constexpr (KEEP) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) bv[v] = bias_of(v);
    }
    float most = 1.f;                                          /* no finite |c| exceeds it */
    if constexpr (BY_SCORE && GROUPS != 0) {
        float b = 0.f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            const float a = fabsf(KEEP ? bv[KEEP ? v : 0] : bias_of(v));
            b = a < INFINITY ? fmaxf(b, a) : b;
        }
        most += warp_max(b);
    }
    const long long step = (long long)gridDim.x * kRouteWarps;
    for (long long t = (long long)blockIdx.x * kRouteWarps + warp; t < n; t += step) {
        const T* row = logits + t * ld;
        float x[VPL];
        unsigned key[VPL];
        LaneRow<T, VPL>::load(row, sh.E, sh.vec, lane, x);
        float mx = 0.f, sum = 1.f, smax = 1.f;
        if (scores) {
            float c[VPL];
            if (softmax) {
                mx = x[0];
#pragma unroll
                for (int v = 1; v < VPL; ++v) mx = fmaxf(mx, x[v]);
                mx = warp_max(mx);
                if (mx == -INFINITY) mx = 0.f;
                sum = 0.f;
#pragma unroll
                for (int v = 0; v < VPL; ++v) { c[v] = exp2_fast((x[v] - mx) * kLog2e); sum += c[v]; }
                sum = warp_sum(sum);
                smax = rcp_fast(sum);
#pragma unroll
                for (int v = 0; v < VPL; ++v) c[v] *= smax;
            } else {
#pragma unroll
                for (int v = 0; v < VPL; ++v) c[v] = rcp_fast(1.f + exp2_fast(x[v] * -kLog2e));
            }
            if constexpr (BY_SCORE) {
#pragma unroll
                for (int v = 0; v < VPL; ++v) {
                    c[v] += KEEP ? bv[KEEP ? v : 0] : bias_of(v);
                    key[v] = x[v] == -INFINITY ? 0u : key_of(c[v]);
                }
            }
        }
        if constexpr (!BY_SCORE) {
#pragma unroll
            for (int v = 0; v < VPL; ++v) key[v] = key_of(x[v]);
        }
        /* Error bounds of c, in units of 2^-24.  e^d from exp2_fast is off by 4 + 2.3 |d| of itself: the instruction,
         * and for a softmax value the roundings of d = x - mx, of its product with log2 e and of that constant (1.3 |d|
         * for a sigmoid, whose argument is exact).
         * A sigmoid turns that into s (1 - s) of it, under 1.1, and adds 2 s for the reciprocal and s for the sum: 4.1.
         * A softmax value e / sum <= smax is off by 4 smax for e (the largest of e^d (4 + 2.3 |d|)) and smax for the
         * product.  The sum's error is shared by all of the row's values and moves a difference of two by no more than
         * its share of smax: VPL + 4 for VPL - 1 additions in a lane and 5 between lanes, the mean of the exponentials'
         * errors, 4 + 2.3 ln E (the mean of |d| is an entropy, ln E at most), and 2 for the reciprocal.  Two values:
         * VPL + 20 + 2.3 ln E, 29 for one expert a lane, 41 for 8, 68 for 32; the VPL + 40 below is above it for all.
         * Relative to a value alone, 5 + 2.3 |d| and the shared part come to under 2^-15 wherever e^d does not
         * underflow.  Adding the bias rounds by |c|. */
        constexpr float kSoftmaxTol = (VPL + 40) * 0x1.0p-24f;
        auto near = [&](float a, float b) {
            const float tol = bias ? (softmax ? kSoftmaxTol : 0x1.4p-21f) * smax + 0x1.1p-24f * (fabsf(a) + fabsf(b))
                                   : 0x1.0p-15f * (fabsf(a) + fabsf(b)) + 1e-37f;
            return !(a - b > tol);
        };
        /* A group's value may be the sum of two c of opposite signs: twice the bound, and roundings (of both and of
         * the sum) that are relative to the largest |c|, not to the sum. */
        auto near_groups = [&](float a, float b) {
            return bias ? !(a - b > (softmax ? 2.f * kSoftmaxTol * smax : 0x1.4p-20f) + 0x1.0p-21f * most) : near(a, b);
        };
        bool slow = false;                                         /* the groups are not certain */
        if constexpr (GROUPS != 0) {
            unsigned gk;
            bool in;
            const int log = GROUPS == 1 ? sh.log_g : sh.log_l;
            if constexpr (GROUPS == 1) {
                unsigned a = 0u, b = 0u;
#pragma unroll
                for (int v = 0; v < VPL; ++v) {
                    b = max(b, min(a, key[v]));
                    a = max(a, key[v]);
                }
                for (int o = (1 << log) >> 1; o > 0; o >>= 1) {
                    const unsigned a2 = __shfl_xor_sync(FULL, a, o), b2 = __shfl_xor_sync(FULL, b, o);
                    b = max(min(a, a2), max(b, b2));
                    a = max(a, a2);
                }
                gk = group_of_two(a, b, sh.group_score);
                in = group_kept(gk, sh, log, lane);
#pragma unroll
                for (int v = 0; v < VPL; ++v)
                    key[v] = !in ? 0u : by_logit_after ? key_of(x[v]) : key[v];
            } else {
#pragma unroll
                for (int v = 0; v < VPL; ++v)
                    if (VPL * lane + v < sh.E) keys32[VPL * lane + v] = key[v];
                __syncwarp();
                gk = group_key(keys32, sh, lane);
                in = group_kept(gk, sh, log, lane);
                const unsigned kept = __ballot_sync(FULL, in);
#pragma unroll
                for (int v = 0; v < VPL; ++v) {
                    const unsigned g = min(31u, ((unsigned)(VPL * lane + v) * sh.gmul >> 20) << log);
                    if (!((kept >> g) & 1u) || VPL * lane + v >= sh.E) key[v] = 0u;
                    else if (by_logit_after) key[v] = key_of(x[v]);
                }
                __syncwarp();
            }
            if constexpr (BY_SCORE) {                              /* the groups on both sides of the cut */
                const bool there = (lane >> log) < sh.G;
                const unsigned lo = __reduce_min_sync(FULL, in ? gk : 0xffffffffu);
                const unsigned hi = __reduce_max_sync(FULL, there && !in ? gk : 0u);
                slow = live(hi) && near_groups(of_key(lo), of_key(hi));
            }
        }
        int mine;
        unsigned mykey;
        top_keys(key, sh.k + (BY_SCORE && bias && sh.k < 32 ? 1 : 0), route_cand[warp], lane, mykey, mine);
        float xi;
        if constexpr (BY_SCORE) {
            bool close = false;                                    /* this slot and the next */
            if (bias) {
                const unsigned nk = __shfl_down_sync(FULL, mykey, 1);
                close = lane < sh.k && lane < 31 && live(nk) && near(of_key(mykey), of_key(nk));
            }
            bool whole = slow || (bias && sh.k == 32);
            if (__any_sync(FULL, close && lane == sh.k - 1)) {
                /* the last slot may tie with the first loser: another that is near it is no higher only where
                 * the bias is the same and the logit no higher */
                const unsigned tk = __shfl_sync(FULL, mykey, sh.k - 1);
                const int tj = __shfl_sync(FULL, mine, sh.k - 1);
                const float tx = to_f(row[tj]), tb = bias[tj];
#pragma unroll
                for (int v = 0; v < VPL; ++v)
                    if (live(key[v]) && key[v] <= tk && near(of_key(tk), of_key(key[v]))) {
                        const int j = VPL * lane + v;
                        if (!(bias[j] == tb && to_f(row[j]) <= tx)) whole = true;
                    }
            }
            if (__any_sync(FULL, whole || close)) mine = slow_choice(row, bias, sh, keys64, lane, mine, close, whole);
            if (lane >= sh.k) mine = -1;
            xi = mine >= 0 ? to_f(row[mine]) : -INFINITY;
        } else {
            xi = mine >= 0 ? of_key(mykey) : -INFINITY;
        }
        const bool valid = mine >= 0;
        float w;
        if (sh.renorm) {
            const float m = slot_max(xi, sh.log_k);
            const float e = valid ? chosen_score(xi, m, softmax) : 0.f;
            const float total = slot_sum(e, sh.log_k);
            w = total == 0.f ? 0.f : __fdividef(e, total);
            if (valid && sum != sum) w = NAN;
        } else {
            w = !valid ? 0.f : softmax ? __fdividef(expf(xi - mx), sum) : __fdividef(1.f, 1.f + expf(-xi));
        }
        if (lane < sh.k) {
            ids[t * sh.k + lane] = mine;
            weights[t * sh.k + lane] = valid ? w * sh.scale : 0.f;
        }
    }
}

/* Gradient of the weights.  With w the weights at scale 1, g the incoming gradient
 * times the scale and G = sum of g w over the slots:
 *   renormalized:  softmax  dl_i = w_i (g_i - G)
 *                  sigmoid  dl_i = w_i (1 - s_i) (g_i - G)      0 off the slots
 *   otherwise:     sigmoid  dl_i = g_i s_i (1 - s_i)            0 off the slots
 *                  softmax  dl_j = s_j ([j chosen] g_j - sum over slots of g s)
 * The first three need the chosen logits only: k_route_grad_slots gives a token
 * 2^log_k lanes, one a slot, and a warp 32 / 2^log_k tokens, whose rows it fills with
 * zeros before the slots' terms go in (ordered by __syncwarp; slots of one expert
 * all write their sum): 4 to 5 us on the device for 30001 x 60.  (A warp a token took
 * 263 instructions a row and 14 us.)  The last form reads and writes whole rows: k_route_grad_whole, one
 * warp a token (22.7 us for 32768 x 256 FP32, whose 67 MB take 10.3 at least). */
template <typename T, typename W>
__global__ void __launch_bounds__(32 * kRouteWarps)
k_route_grad_slots(const T* __restrict__ logits, long long n, long long ld, RouteShape sh, const int* __restrict__ ids,
                   const float* __restrict__ gw, T* __restrict__ out, long long ldg) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool softmax = sh.score == MPK_SCORE_SOFTMAX;
    const int slots = 1 << sh.log_k, tokens = 32 >> sh.log_k;
    const int slot = lane & (slots - 1);
    const int words = sh.E * (int)sizeof(T) / (int)sizeof(W);       /* of a row */
    const long long step = (long long)gridDim.x * kRouteWarps * tokens;
    for (long long t0 = ((long long)blockIdx.x * kRouteWarps + warp) * tokens; t0 < n; t0 += step) {
        const long long t = t0 + (lane >> sh.log_k);
        const bool here = t < n && slot < sh.k;
        int id = here ? ids[t * sh.k + slot] : -1;
        if ((unsigned)id >= (unsigned)sh.E) id = -1;
        const bool valid = id >= 0;
        const float g = valid ? gw[t * sh.k + slot] * sh.scale : 0.f;
        const float xi = valid ? to_f(logits[t * ld + id]) : -INFINITY;
        {
            const int rows = (int)min((long long)tokens, n - t0);
            T* first = out + t0 * ldg;
            const W zero = {};
            if (ldg == sh.E) {
                for (int i = lane; i < rows * words; i += 32) reinterpret_cast<W*>(first)[i] = zero;
            } else {
                for (int r = 0; r < rows; ++r)
                    for (int i = lane; i < words; i += 32) reinterpret_cast<W*>(first + r * ldg)[i] = zero;
            }
        }
        float si = 0.f, left = 1.f, term;                           /* s, 1 - s */
        if (!softmax) {
            si = valid ? __fdividef(1.f, 1.f + expf(-xi)) : 0.f;
            left = valid ? __fdividef(1.f, 1.f + expf(xi)) : 0.f;
        }
        if (sh.renorm) {
            const float m = slot_max(xi, sh.log_k);
            const float e = (!valid || m == -INFINITY) ? 0.f : chosen_score(xi, m, softmax);
            const float total = slot_sum(e, sh.log_k);
            const float w = total == 0.f ? 0.f : __fdividef(e, total);
            const float G = slot_sum(valid ? g * w : 0.f, sh.log_k);
            term = w * left * (g - G);
        } else {
            term = g * si * left;
        }
        float sum = 0.f;                                            /* over the slots of the same expert */
        for (int i = 0; i < sh.k; ++i) {
            const int from = (lane & ~(slots - 1)) + i;
            const int j = __shfl_sync(FULL, id, from);
            const float d = __shfl_sync(FULL, term, from);
            sum += j == id ? d : 0.f;
        }
        __syncwarp();
        if (valid) out[t * ldg + id] = from_f<T>(sum);
    }
}

template <typename T, int VPL>
__global__ void __launch_bounds__(32 * kRouteWarps)
k_route_grad_whole(const T* __restrict__ logits, long long n, long long ld, RouteShape sh, const int* __restrict__ ids,
                   const float* __restrict__ gw, T* __restrict__ out, long long ldg) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long step = (long long)gridDim.x * kRouteWarps;
    for (long long t = (long long)blockIdx.x * kRouteWarps + warp; t < n; t += step) {
        const T* row = logits + t * ld;
        int id = lane < sh.k ? ids[t * sh.k + lane] : -1;
        if ((unsigned)id >= (unsigned)sh.E) id = -1;
        const bool valid = id >= 0;
        const float g = valid ? gw[t * sh.k + lane] * sh.scale : 0.f;
        const float xi = valid ? to_f(row[id]) : -INFINITY;
        float s[VPL], acc[VPL];
        float sum = 0.f;
        LaneRow<T, VPL>::load(row, sh.E, sh.vec, lane, s);
        float mx = s[0];
#pragma unroll
        for (int v = 1; v < VPL; ++v) mx = fmaxf(mx, s[v]);
        mx = warp_max(mx);
        if (mx == -INFINITY) mx = 0.f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) { s[v] = expf(s[v] - mx); sum += s[v]; }
        sum = warp_sum(sum);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;            /* every expert masked: no gradient */
#pragma unroll
        for (int v = 0; v < VPL; ++v) { s[v] *= inv; acc[v] = 0.f; }
        float dot = slot_sum(valid ? g * (expf(xi - mx) * inv) : 0.f, sh.log_k);
        dot = __shfl_sync(FULL, dot, 0);
        for (int i = 0; i < sh.k; ++i) {
            const int j = __shfl_sync(FULL, id, i) - VPL * lane;
            const float d = __shfl_sync(FULL, g, i);
#pragma unroll
            for (int v = 0; v < VPL; ++v) acc[v] += j == v ? d : 0.f;
        }
#pragma unroll
        for (int v = 0; v < VPL; ++v) acc[v] = s[v] * (acc[v] - dot);
        LaneRow<T, VPL>::store(out + t * ldg, sh.E, sh.vec, lane, acc);
    }
}

/* -------------------------------------------------------------- the plan ---- */
/* A stable counting sort.  A block takes a chunk of the entries, each of its
 * warps a contiguous piece, 32 at a time: a ballot for each bit of the expert's
 * number gives the lanes that share it (match_any takes longer the more experts a
 * warp meets), so an entry's rank among its expert's is (entries of earlier blocks) +
 * (of earlier warps) + (of this warp so far) + (lower lanes of its match): no
 * atomics decide an order.  The block sorts its entries in shared memory first and
 * writes each expert's run in one piece.
 *
 * Up to kPlanOne entries one block does everything; above, the blocks' counts
 * (k_plan_count), their prefixes (k_plan_scan) and the placement are three launches,
 * each started as the one before it starts (programmatic dependent launch) and
 * waiting for its end only where it reads its results: the placement ranks its
 * entries meanwhile.  Bound by the latency of those phases, not by memory: 15 us on
 * the device for 1048576 entries of 256 experts.  Chunks of 2048 entries took 18 us
 * there and 7 instead of 9 for 131072; one of 8192 14 and 13. */
constexpr int kPlanThreads = 512, kPlanWarps = kPlanThreads / 32;
constexpr int kPlanPer = 8;                                 /* entries a lane */
constexpr int kPlanChunk = kPlanThreads * kPlanPer;         /* and a block of the multi-block plan */
constexpr int kPlanOne = 2 * kPlanChunk;

__device__ __forceinline__ void next_launch_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

/* A word that an earlier launch may write while this kernel runs: read where it stands, behind wait_for_last_launch
 * (no read-only load, none moved before the wait). */
__device__ __forceinline__ int waited_for(const int* p) { return *static_cast<const volatile int*>(p); }

__device__ __forceinline__ int plan_id(const int* ids, long long i, long long end, int E) {
    const int a = i < end ? ids[i] : -1;
    return (unsigned)a < (unsigned)E ? a : -1;
}

/* The lanes that have a's expert, `bits` bits of which tell experts apart; any for
 * a < 0. */
__device__ __forceinline__ unsigned same_expert(int a, int bits) {
    unsigned m = __ballot_sync(FULL, a >= 0);
    for (int b = 0; b < bits; ++b) {
        const bool one = (a >> b) & 1;
        const unsigned v = __ballot_sync(FULL, one);
        m &= one ? v : ~v;
    }
    return m;
}

/* Exclusive scan of one int per thread over the block; tot receives the total. */
__device__ __forceinline__ int block_scan(int v, int* part, int& tot) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(FULL, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) part[w] = incl;
    __syncthreads();
    int run = 0;
    tot = 0;
#pragma unroll
    for (int q = 0; q < kPlanWarps; ++q) {
        if (q < w) run += part[q];
        tot += part[q];
    }
    __syncthreads();
    return run + incl - v;
}

/* Placement of one chunk.  work: NULL when the chunk is everything, else the
 * scanned counts, work[e * B + b] rows of expert e before block b and totals
 * behind them. */
template <int PER>
__global__ void __launch_bounds__(kPlanThreads)
k_plan(const int* __restrict__ ids, long long m, int E, const int* work, int* __restrict__ offsets,
       int* __restrict__ order, int* __restrict__ pos) {
    constexpr int CHUNK = kPlanThreads * PER;
    extern __shared__ int plan_sm[];
    __shared__ int part[kPlanWarps];
    int* cnt = plan_sm;                          /* kPlanWarps x E: counts, then prefixes over the warps */
    int* first = cnt + kPlanWarps * E;           /* E: sorted row of the chunk's first entry of each expert */
    int* local = first + E;                      /* E: the same inside the chunk */
    int* entry = local + E;                      /* CHUNK: the chunk's entries, sorted */
    unsigned short* owner = reinterpret_cast<unsigned short*>(entry + CHUNK);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int B = gridDim.x, bits = 32 - __clz(E - 1);
    const long long lo = (long long)blockIdx.x * CHUNK + w * (32 * PER);
    int a[PER], rank[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) a[i] = plan_id(ids, lo + 32 * i + lane, m, E);
    for (int i = threadIdx.x; i < kPlanWarps * E; i += kPlanThreads) cnt[i] = 0;
    __syncthreads();
    int* mine = cnt + w * E;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const unsigned peers = same_expert(a[i], bits);
        const int old = a[i] >= 0 ? mine[a[i]] : 0;
        rank[i] = old + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (a[i] >= 0 && lane == __ffs(peers) - 1) mine[a[i]] = old + __popc(peers);
        __syncwarp();
    }
    if (work) wait_for_last_launch();
    __syncthreads();
    int gcarry = 0, lcarry = 0;
    for (int e0 = 0; e0 < E; e0 += kPlanThreads) {
        const int e = e0 + threadIdx.x;
        int own = 0;
        if (e < E) {
#pragma unroll
            for (int q = 0; q < kPlanWarps; ++q) {
                const int c = cnt[q * E + e];
                cnt[q * E + e] = own;
                own += c;
            }
        }
        int ltot, gtot;
        const int lbase = lcarry + block_scan(own, part, ltot);
        int gbase = lbase;
        if (work) {
            gbase = gcarry + block_scan(e < E ? waited_for(work + (size_t)E * B + e) : 0, part, gtot);
            gcarry += gtot;
        }
        lcarry += ltot;
        if (e < E) {
            local[e] = lbase;
            first[e] = gbase + (work ? waited_for(work + (size_t)e * B + blockIdx.x) : 0);
            if (blockIdx.x == 0) offsets[e] = gbase;
        }
    }
    const int total = work ? gcarry : lcarry;
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[E] = total;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const long long q = lo + 32 * i + lane;
        int p = -1;
        if (a[i] >= 0) {
            const int r = mine[a[i]] + rank[i];
            p = first[a[i]] + r;
            entry[local[a[i]] + r] = (int)q;
            owner[local[a[i]] + r] = (unsigned short)a[i];
        }
        if (q < m) pos[q] = p;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < lcarry; i += kPlanThreads) {
        const int e = owner[i];
        order[first[e] + (i - local[e])] = entry[i];
    }
    for (long long r = total + (long long)blockIdx.x * kPlanThreads + threadIdx.x; r < m; r += (long long)B * kPlanThreads)
        order[r] = -1;
}

/* This block's entries of each expert, to work[e * B + b]. */
__global__ void __launch_bounds__(kPlanThreads)
k_plan_count(const int* __restrict__ ids, long long m, int E, int* __restrict__ work) {
    extern __shared__ int plan_sm[];
    next_launch_may_start();
    for (int e = threadIdx.x; e < E; e += kPlanThreads) plan_sm[e] = 0;
    __syncthreads();
    int a[kPlanPer];
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i)
        a[i] = plan_id(ids, (long long)blockIdx.x * kPlanChunk + i * kPlanThreads + threadIdx.x, m, E);
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i)
        if (a[i] >= 0) atomicAdd(&plan_sm[a[i]], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kPlanThreads) work[(size_t)e * gridDim.x + blockIdx.x] = plan_sm[e];
}

/* One warp an expert: its counts over the blocks become their exclusive prefix,
 * its total goes behind them. */
__global__ void k_plan_scan(int* work, int E, int B) {
    const int lane = threadIdx.x & 31, e = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    next_launch_may_start();
    wait_for_last_launch();
    if (e >= E) return;
    int* row = work + (size_t)e * B;
    int run = 0;
    for (int b0 = 0; b0 < B; b0 += 32) {
        const int v = b0 + lane < B ? waited_for(row + b0 + lane) : 0;
        int incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(FULL, incl, o);
            if (lane >= o) incl += u;
        }
        if (b0 + lane < B) row[b0 + lane] = run + incl - v;
        run += __shfl_sync(FULL, incl, 31);
    }
    if (lane == 0) work[(size_t)E * B + e] = run;
}

/* ------------------------------------------------------------- host side ---- */

bool route_shape(const mpkRouteParams* p, RouteShape& sh, bool choice) {
    if (!p || p->experts < 1 || p->experts > MPK_MAX_EXPERTS || p->top_k < 1 || p->top_k > MPK_MAX_TOP_K ||
        p->top_k > p->experts || (p->score != MPK_SCORE_SOFTMAX && p->score != MPK_SCORE_SIGMOID) ||
        !std::isfinite(p->scale))
        return false;
    sh = RouteShape{p->experts, p->top_k, p->score, 1, p->experts, 1, MPK_GROUP_MAX, p->renormalize ? 1 : 0, 0, p->scale, 0, 0, -1, 0};
    if (choice) {
        if (p->groups < 1 || p->groups > MPK_MAX_GROUPS || p->experts % p->groups || p->top_groups < 1 ||
            p->top_groups > p->groups || (p->group_score != MPK_GROUP_MAX && p->group_score != MPK_GROUP_TOP2))
            return false;
        sh.G = p->groups;
        sh.gs = p->experts / p->groups;
        sh.top_groups = p->top_groups;
        sh.group_score = p->group_score;
    }
    while ((2 << sh.log_l) * sh.G <= 32) ++sh.log_l;
    while ((1 << sh.log_k) < sh.k) ++sh.log_k;
    /* j * gmul / 2^20 exceeds j / gs by less than j / 2^20 < 1 / gs */
    sh.gmul = ((1u << 20) + sh.gs - 1) / sh.gs;
    return true;
}

/* one warp a token until every SM holds its 16 blocks of four warps */
int route_grid(long long n, int sms) {
    const long long b = (n + kRouteWarps - 1) / kRouteWarps;
    return (int)(b < (long long)sms * 16 ? b : (long long)sms * 16);
}

/* Addresses and row stride let a lane move its VPL elements as whole words. */
template <typename T, int VPL>
bool lane_words(const void* p, long long n, long long ld) {
    constexpr int W = LaneRow<T, VPL>::WORD;
    return reinterpret_cast<uintptr_t>(p) % W == 0 && (n <= 1 || ld * (long long)sizeof(T) % W == 0);
}

template <typename T, int VPL>
cudaError_t run_route(RouteShape sh, const void* logits, long long n, long long ld, const float* bias, int* ids,
                      float* w, int sms, cudaStream_t s) {
    sh.vec = lane_words<T, VPL>(logits, n, ld);
    const int lanes = sh.gs / VPL;
    if (sh.gs % VPL == 0 && (lanes & (lanes - 1)) == 0) {
        sh.log_g = 0;
        while ((1 << sh.log_g) < lanes) ++sh.log_g;
    }
    const bool grouped = sh.G > 1 && sh.top_groups < sh.G;
    const bool by_score = bias || (grouped && sh.group_score == MPK_GROUP_TOP2);
    const size_t smem = (by_score || grouped) ? (size_t)kRouteWarps * sh.E * 8 : 0;
    const auto kern = !grouped ? (by_score ? k_route<T, VPL, true, 0> : k_route<T, VPL, false, 0>)
                    : sh.log_g >= 0 ? (by_score ? k_route<T, VPL, true, 1> : k_route<T, VPL, false, 1>)
                                    : (by_score ? k_route<T, VPL, true, 2> : k_route<T, VPL, false, 2>);
    kern<<<route_grid(n, sms), 32 * kRouteWarps, smem, s>>>(static_cast<const T*>(logits), n, ld, bias, sh, ids, w);
    return cudaGetLastError();
}

template <typename T, int VPL>
cudaError_t run_route_grad(RouteShape sh, const void* logits, long long n, long long ld, const int* ids,
                           const float* gw, void* out, long long ldg, int sms, cudaStream_t s) {
    const T* x = static_cast<const T*>(logits);
    T* o = static_cast<T*>(out);
    if (sh.score == MPK_SCORE_SOFTMAX && !sh.renorm) {
        sh.vec = lane_words<T, VPL>(logits, n, ld) && lane_words<T, VPL>(out, n, ldg);
        k_route_grad_whole<T, VPL><<<route_grid(n, sms), 32 * kRouteWarps, 0, s>>>(x, n, ld, sh, ids, gw, o, ldg);
        return cudaGetLastError();
    }
    const int tokens = 32 >> sh.log_k, grid = route_grid((n + tokens - 1) / tokens, sms);
    /* the widest word that rows are made of */
    const uintptr_t grain = reinterpret_cast<uintptr_t>(out) | (uintptr_t)(sh.E * sizeof(T)) |
                            (n > 1 ? (uintptr_t)ldg * sizeof(T) : 0);
    if (grain % 16 == 0) k_route_grad_slots<T, uint4><<<grid, 32 * kRouteWarps, 0, s>>>(x, n, ld, sh, ids, gw, o, ldg);
    else if (grain % 4 == 0) k_route_grad_slots<T, unsigned><<<grid, 32 * kRouteWarps, 0, s>>>(x, n, ld, sh, ids, gw, o, ldg);
    else k_route_grad_slots<T, unsigned short><<<grid, 32 * kRouteWarps, 0, s>>>(x, n, ld, sh, ids, gw, o, ldg);
    return cudaGetLastError();
}

/* The registers a row takes: 32 * VPL >= experts. */
#define MPK_BY_WIDTH(T, CALL)                                      \
    (sh.E <= 32 ? CALL(T, 1) : sh.E <= 64 ? CALL(T, 2) : sh.E <= 128 ? CALL(T, 4) \
     : sh.E <= 256 ? CALL(T, 8) : sh.E <= 512 ? CALL(T, 16) : CALL(T, 32))
#define MPK_BY_TYPE(CALL)                                          \
    (type == MPK_TYPE_FP32 ? MPK_BY_WIDTH(float, CALL)             \
     : type == MPK_TYPE_FP16 ? MPK_BY_WIDTH(__half, CALL) : MPK_BY_WIDTH(__nv_bfloat16, CALL))

bool type_ok(int type) { return type == MPK_TYPE_FP32 || type == MPK_TYPE_FP16 || type == MPK_TYPE_BF16; }

long long plan_blocks(long long m) { return m <= kPlanOne ? 1 : (m + kPlanChunk - 1) / kPlanChunk; }

/* A launch that may start as the one before it in the stream starts. */
template <typename... P, typename... A>
cudaError_t launch_behind(void (*kern)(P...), int grid, int block, int smem, cudaStream_t s, A... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3((unsigned)block, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, P(args)...);
}

template <int PER>
cudaError_t run_plan(const int* ids, long long m, int E, int B, const int* work, int* offsets, int* order, int* pos,
                     cudaStream_t s) {
    const auto bytes = [](int experts) { return (kPlanWarps + 2) * experts * (int)sizeof(int) + kPlanThreads * PER * 6; };
    const int smem = bytes(E);
    if (smem > 48 * 1024) {
        /* the limit belongs to the kernel, not to this call: every call sets the same */
        const cudaError_t e =
            cudaFuncSetAttribute(k_plan<PER>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes(MPK_MAX_EXPERTS));
        if (e != cudaSuccess) return e;
    }
    if (!work) {
        k_plan<PER><<<B, kPlanThreads, smem, s>>>(ids, m, E, work, offsets, order, pos);
        return cudaGetLastError();
    }
    return launch_behind(k_plan<PER>, B, kPlanThreads, smem, s, ids, m, E, work, offsets, order, pos);
}

}  /* namespace */
}  /* namespace mpk */

using namespace mpk;

extern "C" {

void mpkRouteParamsInit(mpkRouteParams* p) {
    if (!p) return;
    *p = mpkRouteParams{0, 0, MPK_SCORE_SOFTMAX, 1, 1, MPK_GROUP_MAX, 1, 1.0f};
}

mpkStatus mpkRoute(cudaStream_t stream, const mpkRouteParams* p, const void* dLogits, int type, long long n,
                   long long ld, const float* dBias, int* dIds, float* dWeights) {
    RouteShape sh;
    if (!route_shape(p, sh, true) || !type_ok(type) || n < 0 || n > (1LL << 40) || ld < sh.E) return MPK_ERR_INVALID;
    if (n == 0) return MPK_OK;
    if (!dLogits || !dIds || !dWeights) return MPK_ERR_INVALID;
    const int sms = sm_count();
    if (!sms) return MPK_ERR_CUDA;
#define MPK_ROUTE(T, V) run_route<T, V>(sh, dLogits, n, ld, dBias, dIds, dWeights, sms, stream)
    return MPK_BY_TYPE(MPK_ROUTE) == cudaSuccess ? MPK_OK : MPK_ERR_CUDA;
#undef MPK_ROUTE
}

mpkStatus mpkRouteGrad(cudaStream_t stream, const mpkRouteParams* p, const void* dLogits, int type, long long n,
                       long long ld, const int* dIds, const float* dGradWeights, void* dGradLogits, long long ldg) {
    RouteShape sh;
    if (!route_shape(p, sh, false) || !type_ok(type) || n < 0 || n > (1LL << 40) || ld < sh.E || ldg < sh.E)
        return MPK_ERR_INVALID;
    if (n == 0) return MPK_OK;
    if (!dLogits || !dIds || !dGradWeights || !dGradLogits) return MPK_ERR_INVALID;
    const int sms = sm_count();
    if (!sms) return MPK_ERR_CUDA;
#define MPK_ROUTE(T, V) run_route_grad<T, V>(sh, dLogits, n, ld, dIds, dGradWeights, dGradLogits, ldg, sms, stream)
    return MPK_BY_TYPE(MPK_ROUTE) == cudaSuccess ? MPK_OK : MPK_ERR_CUDA;
#undef MPK_ROUTE
}

size_t mpkExpertPlanBytes(long long n, int top_k, int experts) {
    if (n <= 0 || top_k < 1 || experts < 1 || experts > MPK_MAX_EXPERTS || n > (1LL << 30) / top_k) return 0;
    const long long B = plan_blocks(n * top_k);
    return B == 1 ? 0 : (size_t)(experts * B + experts) * sizeof(int);
}

mpkStatus mpkExpertPlan(cudaStream_t stream, const int* dIds, long long n, int top_k, int experts, int* dOffsets,
                        int* dOrder, int* dPos, void* dWork, size_t work_bytes) {
    if (n < 0 || top_k < 1 || experts < 1 || experts > MPK_MAX_EXPERTS || n > ((1LL << 30) - 1) / top_k || !dOffsets)
        return MPK_ERR_INVALID;
    const long long m = n * top_k;
    if (m > 0 && (!dIds || !dOrder || !dPos)) return MPK_ERR_INVALID;
    const size_t need = mpkExpertPlanBytes(n, top_k, experts);
    if (need && (!dWork || work_bytes < need || reinterpret_cast<uintptr_t>(dWork) % sizeof(int))) return MPK_ERR_INVALID;
    const int B = (int)plan_blocks(m);
    int* work = static_cast<int*>(dWork);
    cudaError_t e;
    if (B > 1) {
        k_plan_count<<<B, kPlanThreads, experts * (int)sizeof(int), stream>>>(dIds, m, experts, work);
        e = cudaGetLastError();
        if (e == cudaSuccess) e = launch_behind(k_plan_scan, (experts + 7) / 8, 256, 0, stream, work, experts, B);
        if (e == cudaSuccess) e = run_plan<kPlanPer>(dIds, m, experts, B, work, dOffsets, dOrder, dPos, stream);
    } else if (m <= kPlanThreads) {
        e = run_plan<1>(dIds, m, experts, 1, nullptr, dOffsets, dOrder, dPos, stream);
    } else if (m <= 4 * kPlanThreads) {
        e = run_plan<4>(dIds, m, experts, 1, nullptr, dOffsets, dOrder, dPos, stream);
    } else {
        e = run_plan<kPlanOne / kPlanThreads>(dIds, m, experts, 1, nullptr, dOffsets, dOrder, dPos, stream);
    }
    if (e != cudaSuccess) return MPK_ERR_CUDA;
    return cudaGetLastError() == cudaSuccess ? MPK_OK : MPK_ERR_CUDA;
}

}  /* extern "C" */
