/* experts.cu -- the experts' products and the combination of their rows: C ABI
 * (include/mpkexperts.h), the kernel for layouts the tensor-core kernel
 * (experts_tc.cu) does not take, and the two combine kernels.
 */
#include "experts.cuh"
#include "mpkexperts.h"

#include <atomic>
#include <type_traits>

namespace mpk {
namespace {

constexpr unsigned FULL = 0xffffffffu;

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

/* ------------------------------------------------- products, any layout ---- */

constexpr int GT = 64;                       /* output tile: 64 rows x 64 columns */
constexpr int GC = 16;                       /* contraction step */
constexpr int kAnyThreads = 256;

/* Token row of sorted row r; -1 (read as zeros) where the plan names none. */
__device__ __forceinline__ long long x_row(const ExpertArgs& a, long long r) {
    if (!a.order) return r;
    const int entry = a.order[r];
    return (unsigned)entry < (unsigned long long)a.m ? entry / a.top_k : -1;
}

/* The kernel of odd layouts, 15 to 19 TFLOP/s: its loads are single elements.
 * One 64 x 64 tile of one expert's output a block, operands staged in shared
 * memory 16 deep, 4 x 4 sums a thread.  FWD and GRADX: blockIdx.x counts the row
 * tiles of all experts (their number T is known on the device only; with D rows
 * that no expert owns, T <= (m - D) / 64 + 63 experts / 64, so m / 64 + experts + 1
 * blocks leave at least D / 64 past T, which set those rows to zero); GRADW: blockIdx.x = expert * column tiles + tile. */
template <typename T, int MODE>
__global__ void __launch_bounds__(kAnyThreads) k_experts_any(const ExpertArgs a) {
    __shared__ float sa[GC][GT + 1], sb[GC][GT + 1];
    __shared__ int where[2];
    const int F = MODE == EXP_FWD ? a.width : a.k;
    const int f0 = blockIdx.y * GT;
    const int m = (int)a.m;
    int e, tile;
    if (MODE == EXP_GRADW) {
        const int tiles = (a.width + GT - 1) / GT;
        e = blockIdx.x / tiles;
        tile = blockIdx.x - e * tiles;
    } else {
        if (threadIdx.x < 32) {              /* the expert whose row tiles hold tile blockIdx.x */
            const int lane = threadIdx.x;
            int run = 0, fe = -1, ft = 0;
            for (int e0 = 0; e0 < a.experts && fe < 0; e0 += 32) {
                const int q = e0 + lane;
                const int t = q < a.experts
                    ? (max(expert_start(a.offsets, q + 1, m) - expert_start(a.offsets, q, m), 0) + GT - 1) / GT : 0;
                int incl = t;
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(FULL, incl, o);
                    if (lane >= o) incl += u;
                }
                const unsigned hit = __ballot_sync(FULL, run + incl > (int)blockIdx.x);
                if (hit) {
                    const int l = __ffs(hit) - 1;
                    fe = e0 + l;
                    ft = (int)blockIdx.x - run - __shfl_sync(FULL, incl - t, l);
                }
                run = min(run + __shfl_sync(FULL, incl, 31), 1 << 29);   /* more than any plan's tiles */
            }
            if (lane == 0) { where[0] = fe; where[1] = fe < 0 ? (int)blockIdx.x - run : ft; }
        }
        __syncthreads();
        e = where[0];
        tile = where[1];
    }
    T* out = static_cast<T*>(a.out);
    if (MODE != EXP_GRADW && e < 0) {
        const long long r0 = expert_start(a.offsets, a.experts, m) + (long long)tile * GT;
        for (int i = threadIdx.x; i < GT * GT; i += kAnyThreads) {
            const long long r = r0 + i / GT;
            const int f = f0 + i % GT;
            if (r < m && f < F) out[r * a.ldo + f] = from_f<T>(0.f);
        }
        return;
    }
    const int r0 = expert_start(a.offsets, e, m), r1 = expert_start(a.offsets, e + 1, m);
    const int j0 = tile * GT;                                          /* first output row inside the expert */
    const int J = MODE == EXP_GRADW ? a.width : r1 - r0;
    const int C = MODE == EXP_FWD ? a.k : MODE == EXP_GRADX ? a.width : max(r1 - r0, 0);
    const T* x = static_cast<const T*>(a.x);
    const T* gy = static_cast<const T*>(a.gy);
    const T* w = static_cast<const T*>(a.w) + (long long)e * a.stride_w;
    float acc[4][4] = {};
    const int tf = threadIdx.x & 15, tj = threadIdx.x >> 4;
    for (int c0 = 0; c0 < C; c0 += GC) {
        for (int i = threadIdx.x; i < GC * GT; i += kAnyThreads) {
            /* neighbouring threads read along the operand's contiguous dimension */
            const bool a_c = MODE == EXP_FWD, b_c = MODE != EXP_GRADW;
            {
                const int c = a_c ? i % GC : i / GT, f = a_c ? i / GC : i % GT;
                float v = 0.f;
                if (c0 + c < C && f0 + f < F) {
                    if (MODE == EXP_FWD) v = to_f(w[(long long)(f0 + f) * a.ldw + c0 + c]);
                    else if (MODE == EXP_GRADX) v = to_f(w[(long long)(c0 + c) * a.ldw + f0 + f]);
                    else {
                        const long long q = x_row(a, r0 + c0 + c);
                        if (q >= 0) v = to_f(x[q * a.ldx + f0 + f]);
                    }
                }
                sa[c][f] = v;
            }
            {
                const int c = b_c ? i % GC : i / GT, j = b_c ? i / GC : i % GT;
                float v = 0.f;
                if (c0 + c < C && j0 + j < J) {
                    if (MODE == EXP_FWD) {
                        const long long q = x_row(a, r0 + j0 + j);
                        if (q >= 0) v = to_f(x[q * a.ldx + c0 + c]);
                    } else if (MODE == EXP_GRADX) {
                        v = to_f(gy[(long long)(r0 + j0 + j) * a.ldgy + c0 + c]);
                    } else {
                        v = to_f(gy[(long long)(r0 + c0 + c) * a.ldgy + j0 + j]);
                    }
                }
                sb[c][j] = v;
            }
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < GC; ++c) {
            float va[4], vb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { va[i] = sa[c][tf + 16 * i]; vb[i] = sb[c][tj + 16 * i]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[i][q] = fmaf(va[q], vb[i], acc[i][q]);
        }
        __syncthreads();
    }
    T* base = MODE == EXP_GRADW ? out + (long long)e * a.stride_o : out + (long long)r0 * a.ldo;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int j = j0 + tj + 16 * i, f = f0 + tf + 16 * q;
            if (j < J && f < F) base[(long long)j * a.ldo + f] = from_f<T>(acc[i][q]);
        }
}

template <typename T>
cudaError_t launch_any(const ExpertArgs& a, cudaStream_t s) {
    const int F = a.mode == EXP_FWD ? a.width : a.k;
    const unsigned ft = (unsigned)((F + GT - 1) / GT);
    if (a.mode == EXP_GRADW) {
        const dim3 g((unsigned)a.experts * (unsigned)((a.width + GT - 1) / GT), ft);
        k_experts_any<T, EXP_GRADW><<<g, kAnyThreads, 0, s>>>(a);
    } else {
        const dim3 g((unsigned)(a.m / GT + a.experts + 1), ft);
        if (a.mode == EXP_FWD) k_experts_any<T, EXP_FWD><<<g, kAnyThreads, 0, s>>>(a);
        else k_experts_any<T, EXP_GRADX><<<g, kAnyThreads, 0, s>>>(a);
    }
    return cudaGetLastError();
}

/* ------------------------------------------------- products of few rows ---- */

constexpr int kFewThreads = 256;
constexpr int kFewF = 4;                     /* outputs a warp forms at a time */
constexpr int kFewBlockF = kFewF * kFewThreads / 32;

template <typename T>
__device__ __forceinline__ float2 two_floats(uint32_t u);
template <>
__device__ __forceinline__ float2 two_floats<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
template <>
__device__ __forceinline__ float2 two_floats<__nv_bfloat16>(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}

/* Eight elements from column c of a row; zeros past k, which nothing is read of. */
template <typename T>
__device__ __forceinline__ uint4 eight(const T* row, int c, int k) {
    if (c + 8 <= k) return *reinterpret_cast<const uint4*>(row + c);
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    T* t = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < k) t[i] = row[c + i];
    return u;
}

/* R rows of one expert (from sorted row r, there of them real) times kFewF of its
 * outputs from f: lane l takes elements 8 l ... of every 256.  Rows and outputs
 * that do not exist repeat one that does, so that no load waits on a branch; a row
 * that the plan names no token for reads token 0 and is set to zero at the end. */
template <typename T, int R>
__device__ __forceinline__ void few_rows(const ExpertArgs& a, const T* we, int f, int r, int there, int lane) {
    const T* x[R];
    const T* w[kFewF];
    bool named = true;                       /* the row of this lane's output, lane % R */
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const long long q = x_row(a, r + min(i, there - 1));
        if (lane % R == i) named = q >= 0;
        x[i] = static_cast<const T*>(a.x) + max(q, 0LL) * a.ldx;
    }
#pragma unroll
    for (int j = 0; j < kFewF; ++j) w[j] = we + (long long)min(f + j, a.width - 1) * a.ldw;
    float acc[kFewF][R] = {};
    auto step = [&](const uint4 (&uw)[kFewF], const uint4 (&ux)[R]) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            float2 fx[R];
#pragma unroll
            for (int i = 0; i < R; ++i) fx[i] = two_floats<T>((&ux[i].x)[h]);
#pragma unroll
            for (int j = 0; j < kFewF; ++j) {
                const float2 fw = two_floats<T>((&uw[j].x)[h]);
#pragma unroll
                for (int i = 0; i < R; ++i) acc[j][i] = fmaf(fw.y, fx[i].y, fmaf(fw.x, fx[i].x, acc[j][i]));
            }
        }
    };
    constexpr int U = R <= 2 ? 4 : 2;        /* steps whose loads are in flight together */
    int c = 8 * lane;
    const int whole = a.k / (256 * U) * (256 * U);
    for (; c < whole; c += 256 * U) {
        uint4 uw[U][kFewF], ux[U][R];
#pragma unroll
        for (int t = 0; t < U; ++t) {
#pragma unroll
            for (int j = 0; j < kFewF; ++j) uw[t][j] = __ldcs(reinterpret_cast<const uint4*>(w[j] + c + 256 * t));
#pragma unroll
            for (int i = 0; i < R; ++i) ux[t][i] = *reinterpret_cast<const uint4*>(x[i] + c + 256 * t);
        }
#pragma unroll
        for (int t = 0; t < U; ++t) step(uw[t], ux[t]);
    }
    for (; c < a.k; c += 256) {
        uint4 uw[kFewF], ux[R];
#pragma unroll
        for (int j = 0; j < kFewF; ++j) uw[j] = eight(w[j], c, a.k);
#pragma unroll
        for (int i = 0; i < R; ++i) ux[i] = eight(x[i], c, a.k);
        step(uw, ux);
    }
    float mine = 0.f;                        /* lane j * R + i ends with output j of row i */
#pragma unroll
    for (int j = 0; j < kFewF; ++j)
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float v = acc[j][i];
            for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
            if (lane == j * R + i) mine = v;
        }
    const int j = lane / R, i = lane % R;
    if (j < kFewF && i < there && f + j < a.width)
        static_cast<T*>(a.out)[(long long)(r + i) * a.ldo + f + j] = from_f<T>(named ? mine : 0.f);
}

/* FWD for a handful of rows: bound by reading the chosen experts' matrices once,
 * which many small pieces spread over the SMs better than 128-row tiles do (eight
 * experts of 1536 x 2048 make 96 tiles, 384 blocks here).  blockIdx.y counts the
 * experts that have rows, blockIdx.x their outputs, kFewBlockF a block; four rows
 * at a time share a pass over W. */
template <typename T>
__global__ void __launch_bounds__(kFewThreads, 2) k_experts_few(const ExpertArgs a) {
    __shared__ int found;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = (int)a.m;
    if (warp == 0) {                         /* the blockIdx.y-th expert with rows */
        int seen = 0, e = -1;
        for (int e0 = 0; e0 < a.experts && e < 0; e0 += 32) {
            const int q = e0 + lane;
            const bool some = q < a.experts && expert_start(a.offsets, q + 1, m) > expert_start(a.offsets, q, m);
            unsigned who = __ballot_sync(FULL, some);
            const int more = __popc(who);
            if (seen + more > (int)blockIdx.y) {
                for (int skip = (int)blockIdx.y - seen; skip > 0; --skip) who &= who - 1;
                e = e0 + __ffs(who) - 1;
            }
            seen += more;
        }
        if (lane == 0) found = e;
    }
    __syncthreads();
    const int e = found, f0 = blockIdx.x * kFewBlockF;
    /* rows that no expert owns: this block's outputs of its share */
    for (int r = expert_start(a.offsets, a.experts, m) + (int)blockIdx.y; r < m; r += gridDim.y)
        if ((int)threadIdx.x < kFewBlockF && f0 + (int)threadIdx.x < a.width)
            static_cast<T*>(a.out)[(long long)r * a.ldo + f0 + threadIdx.x] = from_f<T>(0.f);
    if (e < 0) return;
    const int r1 = expert_start(a.offsets, e + 1, m);
    const T* w = static_cast<const T*>(a.w) + (long long)e * a.stride_w;
    const int f = f0 + warp * kFewF;
    if (f >= a.width) return;
    for (int r = expert_start(a.offsets, e, m); r < r1; r += 4) {
        if (r1 - r == 1) few_rows<T, 1>(a, w, f, r, 1, lane);
        else if (r1 - r == 2) few_rows<T, 2>(a, w, f, r, 2, lane);
        else few_rows<T, 4>(a, w, f, r, min(4, r1 - r), lane);
    }
}

template <typename T>
cudaError_t launch_few(const ExpertArgs& a, cudaStream_t s) {
    const dim3 g((unsigned)((a.width + kFewBlockF - 1) / kFewBlockF), (unsigned)(a.m < a.experts ? a.m : a.experts));
    k_experts_few<T><<<g, kFewThreads, 0, s>>>(a);
    return cudaGetLastError();
}

/* ------------------------------------------------------ sorted copy of X ---- */

constexpr int kCopyThreads = 256;

/* out[r] = x[order[r] / top_k] for the *rows sorted rows there are (zeros where the
 * entry names no row), V elements a copy: a warp a row, eight copies in flight a lane.  Bound by memory: 32768 rows of 4096
 * from 8192 tokens take 61 us, 5.5 TB/s. */
template <int V>
__global__ void __launch_bounds__(kCopyThreads)
k_sort_rows(const uint16_t* __restrict__ x, long long ldx, const int* __restrict__ order,
            const int* __restrict__ rows, int top_k, int m, int k, uint16_t* __restrict__ out, long long ldo) {
    using W = typename std::conditional<V == 8, uint4, uint16_t>::type;
    const int lane = threadIdx.x & 31;
    const long long warps = (long long)gridDim.x * (kCopyThreads / 32);
    const int pieces = (k + V - 1) / V;
    for (long long r = (long long)blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5); r < m; r += warps) {
        const int entry = order[r];
        W* dst = reinterpret_cast<W*>(out + r * ldo);
        int c = lane;
        if ((unsigned)entry >= (unsigned)m) {
            if (r < *rows)                                     /* not behind the last routed row */
                for (; c < pieces; c += 32) dst[c] = W{};
            continue;
        }
        const W* src = reinterpret_cast<const W*>(x + (long long)(entry / top_k) * ldx);
        for (; c + 7 * 32 < pieces; c += 8 * 32) {
            W v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = src[c + 32 * i];
#pragma unroll
            for (int i = 0; i < 8; ++i) dst[c + 32 * i] = v[i];
        }
        for (; c < pieces; c += 32) dst[c] = src[c];
    }
}

/* --------------------------------------------------------------- combine ---- */

/* V consecutive elements of a row: as they are loaded, and as floats. */
template <typename T, int V>
struct Pack {
    using Raw = typename std::conditional<V == 1, T, uint4>::type;
    __device__ static __forceinline__ Raw raw(const T* p) { return *reinterpret_cast<const Raw*>(p); }
    __device__ static __forceinline__ void open(const Raw& r, float (&f)[V]) {
        const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_f(t[i]);
    }
    __device__ static __forceinline__ void store(T* p, const float (&f)[V]) {
        Raw r;
        T* t = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = from_f<T>(f[i]);
        *reinterpret_cast<Raw*>(p) = r;
    }
};

constexpr int kCombineThreads = 256;

/* TPR threads (a power of two) share a token's row, kCombineThreads / TPR tokens a
 * block, blockIdx.y the TPR-piece span of the row: one thread a 16-byte piece (V
 * elements).  S slots' pieces are in flight at once and are added in slot order in
 * FP32; every row is read once, every output written once.  Bound by memory: 65536
 * BF16 rows of 2048 into 8192 take 49 us, 6.1 TB/s. */
template <typename T, int V, int S>
__global__ void __launch_bounds__(kCombineThreads)
k_combine(const T* __restrict__ y, long long ldy, const int* __restrict__ pos, const float* __restrict__ weights,
          long long n, int top_k, int width, int log_tpr, T* __restrict__ out, long long ldo) {
    const long long t = ((long long)blockIdx.x << (8 - log_tpr)) + (threadIdx.x >> log_tpr);
    const int c = (int)(((blockIdx.y << log_tpr) + (threadIdx.x & ((1u << log_tpr) - 1u))) * V);
    if (t >= n || c >= width) return;
    const long long m = n * top_k;
    float acc[V] = {};
    for (int s0 = 0; s0 < top_k; s0 += S) {
        typename Pack<T, V>::Raw f[S];
        float wt[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const long long q = t * top_k + s0 + s;
            const int p = s0 + s < top_k ? pos[q] : -1;
            const bool there = p >= 0 && p < m;
            wt[s] = !there ? 0.f : weights ? weights[q] : 1.f;
            f[s] = there ? Pack<T, V>::raw(y + (long long)p * ldy + c) : typename Pack<T, V>::Raw{};
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            float v[V];
            Pack<T, V>::open(f[s], v);
#pragma unroll
            for (int u = 0; u < V; ++u) acc[u] = fmaf(wt[s], v[u], acc[u]);
        }
    }
    Pack<T, V>::store(out + t * ldo + c, acc);
}

/* TPR threads (32 .. 256) a token: for every piece of the token's gradient row the
 * S slots' pieces are read together for the weights' dot products and their
 * gradient pieces written.  The dots are summed per thread over its columns, then
 * over the token's threads in a fixed order.  Bound by memory and, at a block's end,
 * its sums: 20012 FP16 rows of 4096 take 64 us, 5.5 TB/s; one piece in flight a
 * thread instead of U = 2 took 75. */
template <typename T, int V, int S>
__global__ void __launch_bounds__(kCombineThreads)
k_combine_grad(const T* __restrict__ go, long long ldgo, const T* __restrict__ y, long long ldy,
               const int* __restrict__ pos, const int* __restrict__ rows, const float* __restrict__ weights,
               long long n, int top_k, int width, int log_tpr, T* __restrict__ gy, long long ldgy,
               float* __restrict__ gw) {
    constexpr int U = S <= 4 ? 2 : 1;            /* pieces of the row in flight */
    __shared__ float part[kCombineThreads / 32][S];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long m = n * top_k;
    const long long t = ((long long)blockIdx.x << (8 - log_tpr)) + (threadIdx.x >> log_tpr);
    const int tpr = 1 << log_tpr, own = threadIdx.x & (tpr - 1);
    for (int s0 = 0; s0 < top_k; s0 += S) {
        int p[S];
        float wt[S], dot[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const long long q = t * top_k + s0 + s;
            p[s] = t < n && s0 + s < top_k ? pos[q] : -1;
            if (p[s] >= m) p[s] = -1;
            wt[s] = p[s] < 0 ? 0.f : weights ? weights[q] : 1.f;
            dot[s] = 0.f;
        }
        if (t < n)
            for (int c0 = own * V; c0 < width; c0 += U * tpr * V) {
                typename Pack<T, V>::Raw rg[U], f[U][S];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int c = c0 + i * tpr * V;
                    if (c < width) {
                        rg[i] = Pack<T, V>::raw(go + t * ldgo + c);
                        if (gw) {
#pragma unroll
                            for (int s = 0; s < S; ++s)
                                if (p[s] >= 0) f[i][s] = Pack<T, V>::raw(y + (long long)p[s] * ldy + c);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int c = c0 + i * tpr * V;
                    if (c >= width) continue;
                    float g[V];
                    Pack<T, V>::open(rg[i], g);
#pragma unroll
                    for (int s = 0; s < S; ++s)
                        if (p[s] >= 0) {
                            float v[V];
                            if (gw) {
                                Pack<T, V>::open(f[i][s], v);
#pragma unroll
                                for (int u = 0; u < V; ++u) dot[s] = fmaf(g[u], v[u], dot[s]);
                            }
#pragma unroll
                            for (int u = 0; u < V; ++u) v[u] = wt[s] * g[u];
                            Pack<T, V>::store(gy + (long long)p[s] * ldgy + c, v);
                        }
                }
            }
        if (gw) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                float v = dot[s];
                for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
                if (lane == 0) part[warp][s] = v;
            }
            __syncthreads();
            if (own < S && s0 + own < top_k && t < n) {
                float v = 0.f;
                for (int q = 0; q < (tpr >> 5); ++q) v += part[warp + q][own];
                gw[t * top_k + s0 + own] = v;
            }
            __syncthreads();
        }
    }
    /* rows that no expert owns */
    const int valid = *rows;
    const int pieces = (width + V - 1) / V;
    const float zero[V] = {};
    for (long long r = (valid < 0 ? 0 : valid) + (long long)blockIdx.x; r < m; r += gridDim.x)
        for (int c = threadIdx.x; c < pieces; c += kCombineThreads) Pack<T, V>::store(gy + r * ldgy + (long long)c * V, zero);
}

/* ------------------------------------------------------------- host side ---- */

bool half_type(int type) { return type == MPK_TYPE_FP16 || type == MPK_TYPE_BF16; }

bool aligned16(const void* p, long long ld, size_t size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (long long)size % 16 == 0;
}

/* What every product needs of its sizes; the gathers' entry index and all row
 * numbers fit 32 bits. */
bool shape_ok(int type, long long m, int experts, int width, int k, bool gather, int top_k) {
    return half_type(type) && m >= 0 && m < (1LL << 30) && experts >= 1 && experts <= MPK_MAX_EXPERTS && width >= 1 &&
           width <= (1 << 20) && k >= 1 && k <= (1 << 20) && (!gather || (top_k >= 1 && m % top_k == 0));
}

/* Row stride of the sorted copy of gathered rows: 16-byte steps. */
long long copy_ld(int k) { return ((long long)k + 7) / 8 * 8; }

size_t copy_bytes(int mode, long long m, int experts, int k) {
    return mode == EXP_FWD && experts_few_rows(m, experts) ? 0 : (size_t)m * copy_ld(k) * 2;
}

/* Up to so many rows the product is a pass over the chosen matrices by plain loads
 * (k_experts_few).  Measured against the 32-row tiles, 64 experts of 1024 x 2048:
 * 16 rows 12 : 20 us, 64 rows 28 : 33 us, 128 rows 45 : 44 us; 8 experts of 1536 x
 * 2048: 16 rows 13 : 18 us, 32 rows 21 : 18 us.  These are even loads.  All rows on
 * one expert walk its matrix once for every four: 64 rows on one of 64 experts of
 * 1024 x 2048 take 74 us in a whole call where 66, on tiles, take 19; the counts are
 * on the device, so the choice cannot see it. */
long long few_limit(int experts) { return experts < 16 ? 16 : experts; }

/* With a sorted copy the product sees plain sorted rows; the tiled kernel gathers
 * for itself and takes none. */
mpkStatus run_product(ExpertArgs& a, void* work, cudaStream_t s) {
    a.sms = sm_count();
    if (!a.sms) return MPK_ERR_CUDA;
    if (a.mode == EXP_FWD && a.m <= few_limit(a.experts) && experts_tc_ok(a))
        return (a.bf16 ? launch_few<__nv_bfloat16>(a, s) : launch_few<__half>(a, s)) == cudaSuccess ? MPK_OK : MPK_ERR_CUDA;
    ExpertArgs sorted = a;
    if (a.order && copy_bytes(a.mode, a.m, a.experts, a.k)) {
        sorted.x = work;
        sorted.ldx = copy_ld(a.k);
        sorted.order = nullptr;
    }
    if (!experts_tc_ok(sorted))
        return (a.bf16 ? launch_any<__nv_bfloat16>(a, s) : launch_any<__half>(a, s)) == cudaSuccess ? MPK_OK : MPK_ERR_CUDA;
    if (a.order && !sorted.order) {
        const long long rows8 = (a.m + kCopyThreads / 32 - 1) / (kCopyThreads / 32), most = (long long)a.sms * 8;
        const int grid = (int)(rows8 < most ? rows8 : most);
        const uint16_t* x = static_cast<const uint16_t*>(a.x);
        uint16_t* out = static_cast<uint16_t*>(work);
        const long long xrows = a.m / a.top_k;
        if (a.k % 8 == 0 && aligned16(x, xrows > 1 ? a.ldx : 8, 2))
            k_sort_rows<8><<<grid, kCopyThreads, 0, s>>>(x, a.ldx, a.order, a.offsets + a.experts, a.top_k, (int)a.m,
                                                           a.k, out, sorted.ldx);
        else
            k_sort_rows<1><<<grid, kCopyThreads, 0, s>>>(x, a.ldx, a.order, a.offsets + a.experts, a.top_k, (int)a.m,
                                                           a.k, out, sorted.ldx);
        if (cudaGetLastError() != cudaSuccess) return MPK_ERR_CUDA;
    }
    return launch_experts_tc(sorted, s) == cudaSuccess ? MPK_OK : MPK_ERR_CUDA;
}

/* A call's scratch: none asked for, or enough of it on a 16-byte boundary. */
bool work_ok(size_t need, const void* work, size_t bytes) {
    return need == 0 || (work && bytes >= need && reinterpret_cast<uintptr_t>(work) % 16 == 0);
}

/* Threads a row (log2): a power of two up to the block that covers the row's pieces. */
int log_threads(int pieces, int least) {
    int l = least;
    while (l < 8 && (1 << l) < pieces) ++l;
    return l;
}

template <typename T, int V, int S>
cudaError_t start_combine(const T* y, long long ldy, const int* pos, const float* weights, long long n, int top_k,
                          int width, T* out, long long ldo, cudaStream_t s) {
    const int pieces = (width + V - 1) / V, l = log_threads(pieces, 0);
    const long long tokens = kCombineThreads >> l;
    const dim3 grid((unsigned)((n + tokens - 1) / tokens), (unsigned)((pieces + (1 << l) - 1) >> l));
    k_combine<T, V, S><<<grid, kCombineThreads, 0, s>>>(y, ldy, pos, weights, n, top_k, width, l, out, ldo);
    return cudaGetLastError();
}

template <typename T>
cudaError_t run_combine(const void* y, long long ldy, const int* pos, const float* weights, long long n, int top_k,
                        int width, void* out, long long ldo, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = width % V == 0 && aligned16(y, ldy, sizeof(T)) && aligned16(out, ldo, sizeof(T));
    const T* py = static_cast<const T*>(y);
    T* po = static_cast<T*>(out);
    if (!vec) return start_combine<T, 1, 8>(py, ldy, pos, weights, n, top_k, width, po, ldo, s);
    return top_k <= 4 ? start_combine<T, V, 4>(py, ldy, pos, weights, n, top_k, width, po, ldo, s)
                      : start_combine<T, V, 8>(py, ldy, pos, weights, n, top_k, width, po, ldo, s);
}

template <typename T, int V, int S>
cudaError_t start_combine_grad(const T* go, long long ldgo, const T* y, long long ldy, const int* pos, const int* rows,
                               const float* weights, long long n, int top_k, int width, T* gy, long long ldgy,
                               float* gw, cudaStream_t s) {
    const int l = log_threads((width + V - 1) / V, 5);
    const long long tokens = kCombineThreads >> l;
    k_combine_grad<T, V, S><<<(unsigned)((n + tokens - 1) / tokens), kCombineThreads, 0, s>>>(
        go, ldgo, y, ldy, pos, rows, weights, n, top_k, width, l, gy, ldgy, gw);
    return cudaGetLastError();
}

template <typename T>
cudaError_t run_combine_grad(const void* go, long long ldgo, const void* y, long long ldy, const int* pos,
                             const int* rows, const float* weights, long long n, int top_k, int width, void* gy,
                             long long ldgy, float* gw, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = width % V == 0 && aligned16(go, ldgo, sizeof(T)) && (!gw || aligned16(y, ldy, sizeof(T))) &&
                     aligned16(gy, ldgy, sizeof(T));
    const T *pg = static_cast<const T*>(go), *py = static_cast<const T*>(y);
    T* po = static_cast<T*>(gy);
    if (!vec)
        return start_combine_grad<T, 1, 8>(pg, ldgo, py, ldy, pos, rows, weights, n, top_k, width, po, ldgy, gw, s);
    return top_k <= 4
        ? start_combine_grad<T, V, 4>(pg, ldgo, py, ldy, pos, rows, weights, n, top_k, width, po, ldgy, gw, s)
        : start_combine_grad<T, V, 8>(pg, ldgo, py, ldy, pos, rows, weights, n, top_k, width, po, ldgy, gw, s);
}

bool combine_ok(int type, long long n, int top_k, int width) {
    return (type == MPK_TYPE_FP32 || half_type(type)) && n >= 0 && top_k >= 1 && top_k <= 1024 &&
           n <= ((1LL << 30) - 1) / top_k && width >= 1 && width <= (1 << 20);
}

}  /* namespace */

int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev >= 0 && dev < 64 && (sms = known[dev].load(std::memory_order_relaxed)) > 0) return sms;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev >= 0 && dev < 64) known[dev].store(sms, std::memory_order_relaxed);
    return sms;
}

}  /* namespace mpk */

using namespace mpk;

extern "C" {

size_t mpkExpertGemmBytes(int grad_w, long long m, int experts, int k) {
    if (m <= 0 || m >= (1LL << 30) || experts < 1 || k < 1 || k > (1 << 20)) return 0;
    return copy_bytes(grad_w ? EXP_GRADW : EXP_FWD, m, experts, k);
}

mpkStatus mpkExpertGemm(cudaStream_t stream, int type, const void* dX, long long ldx, const void* dW, long long ldw,
                        long long strideW, const int* dOffsets, const int* dOrder, int top_k, long long m,
                        int experts, int width, int k, void* dY, long long ldy, void* dWork, size_t work_bytes) {
    if (!shape_ok(type, m, experts, width, k, dOrder != nullptr, top_k) || ldx < k || ldw < k || ldy < width ||
        (experts > 1 && strideW < (long long)(width - 1) * ldw + k))
        return MPK_ERR_INVALID;
    if (m == 0) return MPK_OK;
    if (!dX || !dW || !dOffsets || !dY ||
        (dOrder && !work_ok(copy_bytes(EXP_FWD, m, experts, k), dWork, work_bytes)))
        return MPK_ERR_INVALID;
    ExpertArgs a{EXP_FWD, type == MPK_TYPE_BF16, dX, ldx, nullptr, 0, dW, ldw, strideW, dOffsets, dOrder, top_k,
                 m, experts, width, k, dY, ldy, 0, 0};
    return run_product(a, dWork, stream);
}

mpkStatus mpkExpertGemmGradX(cudaStream_t stream, int type, const void* dGY, long long ldgy, const void* dW,
                             long long ldw, long long strideW, const int* dOffsets, long long m, int experts,
                             int width, int k, void* dGX, long long ldgx) {
    if (!shape_ok(type, m, experts, width, k, false, 1) || ldgy < width || ldw < k || ldgx < k ||
        (experts > 1 && strideW < (long long)(width - 1) * ldw + k))
        return MPK_ERR_INVALID;
    if (m == 0) return MPK_OK;
    if (!dGY || !dW || !dOffsets || !dGX) return MPK_ERR_INVALID;
    ExpertArgs a{EXP_GRADX, type == MPK_TYPE_BF16, nullptr, 0, dGY, ldgy, dW, ldw, strideW, dOffsets, nullptr, 1,
                 m, experts, width, k, dGX, ldgx, 0, 0};
    return run_product(a, nullptr, stream);
}

mpkStatus mpkExpertGemmGradW(cudaStream_t stream, int type, const void* dGY, long long ldgy, const void* dX,
                             long long ldx, const int* dOffsets, const int* dOrder, int top_k, long long m,
                             int experts, int width, int k, void* dGW, long long ldw, long long strideW, void* dWork,
                             size_t work_bytes) {
    if (!shape_ok(type, m, experts, width, k, dOrder != nullptr, top_k) || ldgy < width || ldx < k || ldw < k ||
        (experts > 1 && strideW < (long long)(width - 1) * ldw + k))
        return MPK_ERR_INVALID;
    if ((m > 0 && (!dGY || !dX)) || !dOffsets || !dGW ||
        (dOrder && !work_ok(copy_bytes(EXP_GRADW, m, experts, k), dWork, work_bytes)))
        return MPK_ERR_INVALID;
    ExpertArgs a{EXP_GRADW, type == MPK_TYPE_BF16, dX, ldx, dGY, ldgy, nullptr, 0, 0, dOffsets, dOrder, top_k,
                 m, experts, width, k, dGW, ldw, strideW, 0};
    return run_product(a, dWork, stream);
}

mpkStatus mpkExpertCombine(cudaStream_t stream, int type, const void* dY, long long ldy, const int* dPos,
                           const float* dWeights, long long n, int top_k, int width, void* dOut, long long ldo) {
    if (!combine_ok(type, n, top_k, width) || ldy < width || ldo < width) return MPK_ERR_INVALID;
    if (n == 0) return MPK_OK;
    if (!dY || !dPos || !dOut) return MPK_ERR_INVALID;
    const cudaError_t e =
        type == MPK_TYPE_FP32 ? run_combine<float>(dY, ldy, dPos, dWeights, n, top_k, width, dOut, ldo, stream)
        : type == MPK_TYPE_FP16 ? run_combine<__half>(dY, ldy, dPos, dWeights, n, top_k, width, dOut, ldo, stream)
        : run_combine<__nv_bfloat16>(dY, ldy, dPos, dWeights, n, top_k, width, dOut, ldo, stream);
    return e == cudaSuccess ? MPK_OK : MPK_ERR_CUDA;
}

mpkStatus mpkExpertCombineGrad(cudaStream_t stream, int type, const void* dGOut, long long ldgo, const void* dY,
                               long long ldy, const int* dPos, const int* dRows, const float* dWeights, long long n,
                               int top_k, int width, void* dGY, long long ldgy, float* dGWeights) {
    if (!combine_ok(type, n, top_k, width) || ldgo < width || (dGWeights && ldy < width) || ldgy < width)
        return MPK_ERR_INVALID;
    if (n == 0) return MPK_OK;
    if (!dGOut || (dGWeights && !dY) || !dPos || !dRows || !dGY) return MPK_ERR_INVALID;
    const cudaError_t e =
        type == MPK_TYPE_FP32 ? run_combine_grad<float>(dGOut, ldgo, dY, ldy, dPos, dRows, dWeights, n, top_k, width,
                                                        dGY, ldgy, dGWeights, stream)
        : type == MPK_TYPE_FP16 ? run_combine_grad<__half>(dGOut, ldgo, dY, ldy, dPos, dRows, dWeights, n, top_k,
                                                           width, dGY, ldgy, dGWeights, stream)
        : run_combine_grad<__nv_bfloat16>(dGOut, ldgo, dY, ldy, dPos, dRows, dWeights, n, top_k, width, dGY, ldgy,
                                          dGWeights, stream);
    return e == cudaSuccess ? MPK_OK : MPK_ERR_CUDA;
}

}  /* extern "C" */
