/* mpkexperts.h -- rows routed to experts: scores, plan, products, combination.
 *
 * The trained counterpart of the k-means steps: where mpkAssign sends a row to
 * its nearest centre, mpkRoute sends a token to the top_k best of E experts by
 * learned scores; where mpkUpdate sorts rows by label and sums them,
 * mpkExpertPlan sorts the routed rows by expert, mpkExpertGemm multiplies every
 * row with its expert's matrix, and mpkExpertCombine sums a token's rows back.
 * Each differentiable step has its gradient beside it.  No counterpart in the
 * reference (CornellHPC/mpkmeans has no routing).
 *
 * Conventions.  n tokens, top_k slots each, m = n * top_k routed rows; entry
 * t * top_k + s is slot s of token t.  All pointers named dX are device pointers
 * of the current device, owned by the caller; work runs on `stream`, is only
 * enqueued (no synchronisation, no allocation, no state kept between calls) and
 * can be captured into a CUDA graph (after one call of the same sizes outside a
 * capture, which loads the kernels).  Outputs and scratch overlap nothing else.
 * Leading dimensions (ld...) count elements.
 * A call with n = 0 (or m = 0) writes only what its comment says.  Bad arguments
 * return MPK_ERR_INVALID before anything is enqueued.  The tensor-core products'
 * waits are bounded (4 s): one that runs out ends the kernel with its output
 * incomplete and sets the status word of mpkDebugExpertStatus
 * (mpkmeans_debug.h). */
#ifndef MPKEXPERTS_B200_H
#define MPKEXPERTS_B200_H

#include <stddef.h>

#include <cuda_runtime_api.h>

#include "mpkmeans.h"

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif
#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the matrices. */
typedef enum {
    MPK_TYPE_FP32 = 0,
    MPK_TYPE_FP16 = 1,
    MPK_TYPE_BF16 = 2
} mpkType;

typedef enum {
    MPK_SCORE_SOFTMAX = 0,
    MPK_SCORE_SIGMOID = 1
} mpkScore;

/* How a group of experts is scored: its best choice value, or the sum of its
 * two best. */
typedef enum {
    MPK_GROUP_MAX = 0,
    MPK_GROUP_TOP2 = 1
} mpkGroupScore;

#define MPK_MAX_EXPERTS 1024
#define MPK_MAX_TOP_K 32
#define MPK_MAX_GROUPS 32

/* experts     1 .. MPK_MAX_EXPERTS
 * top_k       1 .. min(MPK_MAX_TOP_K, experts)
 * score       mpkScore: s = softmax of the row's logits, or their sigmoid
 * groups      1 .. MPK_MAX_GROUPS, divides experts: consecutive experts form a
 *             group; 1: no groups
 * top_groups  1 .. groups: experts of the best top_groups groups are eligible
 * group_score mpkGroupScore
 * renormalize non-zero: a token's weights are divided by their sum
 * scale       multiplies the weights (finite) */
typedef struct {
    int   experts;
    int   top_k;
    int   score;
    int   groups;
    int   top_groups;
    int   group_score;
    int   renormalize;
    float scale;
} mpkRouteParams;

/* softmax, one group, renormalized, scale 1; experts and top_k 0 (to be set). */
void mpkRouteParamsInit(mpkRouteParams* p);

/* dLogits: n x experts of `type`, row stride ld.  With s the scores and c = s +
 * dBias (dBias: `experts` floats or NULL; it steers the choice, not the weights)
 * the top_k eligible experts by c are chosen, ties to the lowest index, and
 * written in that order:
 *   dIds     n x top_k int32
 *   dWeights n x top_k FP32: scale * s_i, or scale * s_i / sum of the chosen s.
 * An expert whose logit or bias is -inf is masked: it is never chosen.  Slots
 * that no expert is left for hold id -1 and weight 0; chosen scores that are all
 * zero (sigmoids of logits below -745) give weights of 0.  Logits are compared
 * where the order of c is theirs (no bias, groups by their maximum); elsewhere the
 * choice is the one that c in FP64 makes, values that FP64 rounds to one another
 * being ties: FP32 scores that lie within their error bound of one another are
 * compared again in FP64 (with a bias and top_k = 32 all rows are, which takes three
 * times as long as top_k = 31).  A row with a NaN logit (or +inf, under softmax)
 * gets NaN weights and ids inside [-1, experts) that mean nothing. */
mpkStatus mpkRoute(cudaStream_t stream, const mpkRouteParams* p, const void* dLogits, int type, long long n,
                   long long ld, const float* dBias, int* dIds, float* dWeights);

/* Gradient of the weights with respect to the logits (the choice is constant):
 * dGradLogits (n x experts of `type`, row stride ldg; every entry written) from
 * dGradWeights (n x top_k FP32) and the ids of mpkRoute.  Ids outside [0,
 * experts) take no part.  groups, top_groups and group_score are not read. */
mpkStatus mpkRouteGrad(cudaStream_t stream, const mpkRouteParams* p, const void* dLogits, int type, long long n,
                       long long ld, const int* dIds, const float* dGradWeights, void* dGradLogits, long long ldg);

/* Sorts the m = n * top_k entries of dIds by expert, entries of one expert in
 * ascending order.  Ids outside [0, experts) are dropped.
 *   dOffsets experts + 1: expert e owns sorted rows [dOffsets[e], dOffsets[e+1])
 *   dOrder   m: entry of each sorted row; -1 from dOffsets[experts] on
 *   dPos     m: sorted row of each entry; -1 for dropped entries
 * dWork: mpkExpertPlanBytes bytes of scratch (may be NULL when that is 0).
 * m < 2^30, experts 1 .. MPK_MAX_EXPERTS.  dOffsets is written for n = 0 too. */
size_t mpkExpertPlanBytes(long long n, int top_k, int experts);
mpkStatus mpkExpertPlan(cudaStream_t stream, const int* dIds, long long n, int top_k, int experts, int* dOffsets,
                        int* dOrder, int* dPos, void* dWork, size_t work_bytes);

/* Products of the sorted rows with their experts' matrices (FP16 or BF16, FP32
 * accumulation, one rounding at the end).  dW: experts matrices of width x k,
 * row stride ldw, strideW apart.
 *   mpkExpertGemm:      dY[r] = W_e X[r],          dY m x width (ldy)
 *   mpkExpertGemmGradX: dGX[r] = W_e^T dGY[r],     dGX m x k (ldgx)
 *   mpkExpertGemmGradW: dGW_e = sum_r GY[r] X[r]^T, dGW experts x (width x k)
 * for the rows r of every expert e.  X[r] is row r of dX when dOrder is NULL
 * (dX has m rows) and row dOrder[r] / top_k of dX (n = m / top_k token rows)
 * otherwise, zeros where dOrder[r] is none of the m entries.  Rows of dY and dGX that no expert owns ([dOffsets[experts], m)) are
 * set to zero; an expert without rows gets a zero gradient.  Nothing past row m
 * and nothing between a row's end and its stride is written.
 * With dOrder, dWork is scratch of mpkExpertGemmBytes(0 for Gemm, 1 for GradW, ...)
 * bytes on a 16-byte boundary (a sorted copy of the rows of X; 0 where the
 * experts have few rows and the product gathers them itself); without, it is not
 * looked at.
 * width and k in 1 .. 2^20; any alignment of the element type: rows that start
 * on 16-byte boundaries (addresses and strides) run on the tensor cores, and so do
 * gathered ones that are copied first; with others the product takes ten times as
 * long or more (15 to 19 TFLOP/s). */
size_t mpkExpertGemmBytes(int grad_w, long long m, int experts, int k);
mpkStatus mpkExpertGemm(cudaStream_t stream, int type, const void* dX, long long ldx, const void* dW, long long ldw,
                        long long strideW, const int* dOffsets, const int* dOrder, int top_k, long long m,
                        int experts, int width, int k, void* dY, long long ldy, void* dWork, size_t work_bytes);
mpkStatus mpkExpertGemmGradX(cudaStream_t stream, int type, const void* dGY, long long ldgy, const void* dW,
                             long long ldw, long long strideW, const int* dOffsets, long long m, int experts,
                             int width, int k, void* dGX, long long ldgx);
mpkStatus mpkExpertGemmGradW(cudaStream_t stream, int type, const void* dGY, long long ldgy, const void* dX,
                             long long ldx, const int* dOffsets, const int* dOrder, int top_k, long long m,
                             int experts, int width, int k, void* dGW, long long ldw, long long strideW, void* dWork,
                             size_t work_bytes);

/* dOut[t] = sum over slots s of dWeights[t, s] * dY[dPos[t, s]] (n x width of
 * `type`, FP32 sums in slot order); dWeights NULL: weights of 1 (the gradient of
 * gathering the tokens' rows).  Dropped slots add nothing.  dY has m = n * top_k
 * rows; top_k 1 .. 1024. */
mpkStatus mpkExpertCombine(cudaStream_t stream, int type, const void* dY, long long ldy, const int* dPos,
                           const float* dWeights, long long n, int top_k, int width, void* dOut, long long ldo);

/* Its gradients: dGY[dPos[t, s]] = dWeights[t, s] * dGOut[t] and
 * dGWeights[t, s] = <dGOut[t], dY[dPos[t, s]]> (0 for dropped slots).  dRows: the
 * plan's count of sorted rows (dOffsets + experts); rows from there to m are set
 * to zero.  dWeights NULL: weights of 1.  dGWeights NULL: not wanted, and dY is
 * not read (may be NULL). */
mpkStatus mpkExpertCombineGrad(cudaStream_t stream, int type, const void* dGOut, long long ldgo, const void* dY,
                               long long ldy, const int* dPos, const int* dRows, const float* dWeights, long long n,
                               int top_k, int width, void* dGY, long long ldgy, float* dGWeights);

#ifdef __cplusplus
}
#endif
#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#endif /* MPKEXPERTS_B200_H */
