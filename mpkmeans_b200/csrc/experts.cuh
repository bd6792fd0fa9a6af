/* experts.cuh -- interface of the experts' matrix products (experts_tc.cu, experts.cu). */
#pragma once

#include "common.cuh"

namespace mpk {

/* What a product computes; F is the output's contiguous dimension, J its rows:
 *   FWD    out[r][f = width]  = sum_k  W_e[f][k] X[r][k]
 *   GRADX  out[r][f = k]      = sum_n  W_e[n][f] GY[r][n]
 *   GRADW  out_e[j = n][f = k] = sum_r X[r][f] GY[r][j] */
enum : int { EXP_FWD = 0, EXP_GRADX = 1, EXP_GRADW = 2 };

struct ExpertArgs {
    int mode;
    bool bf16;
    const void* x;            /* FWD, GRADW: rows of X (tokens with order, else sorted) */
    long long ldx;
    const void* gy;           /* GRADX, GRADW: sorted rows of the output's gradient */
    long long ldgy;
    const void* w;            /* FWD, GRADX */
    long long ldw, stride_w;
    const int* offsets;
    const int* order;         /* NULL: X is sorted */
    int top_k;
    long long m;
    int experts, width, k;
    void* out;
    long long ldo, stride_o;  /* GRADW: stride_o between experts */
    int sms;
};

/* Whether the average expert has so few rows that reading W bounds the product:
 * such calls gather rows in the product's kernel; all others, and every gradient
 * of the weights, take X sorted. */
bool experts_few_rows(long long m, int experts);
/* Whether the operands have the layout the tensor-core kernel takes. */
bool experts_tc_ok(const ExpertArgs& a);
cudaError_t launch_experts_tc(const ExpertArgs& a, cudaStream_t s);

/* Multiprocessors of the current device, 0 on an error; looked up once a device. */
int sm_count();

/* Sorted row range of expert e, clamped to the rows there are. */
__device__ __forceinline__ int expert_start(const int* offsets, int e, int m) {
    const int o = offsets[e];
    return o < 0 ? 0 : (o > m ? m : o);
}

}  /* namespace mpk */
