/*
 * What the kernels of the linear layer and of the products by expert share: the
 * arguments of a product C[m][n] = sum_k A(m, k) B(n, k) with its epilogue, the
 * activations, and the epilogue itself on eight consecutive columns of a row.
 */
#ifndef ESHKOL_HIP_LINEAR_ARGS_H
#define ESHKOL_HIP_LINEAR_ARGS_H

#include "layer_common.h"

/* How an operand lies in memory: its rows (m or n) apart and k contiguous, or k
 * apart and the rows contiguous. */
enum { ROWS_K = 0, K_ROWS = 1 };
/* What the groups of experts cut: nothing, the rows of A and C, or the contraction. */
enum { GROUP_NONE = 0, GROUP_ROWS = 1, GROUP_K = 2 };

struct LinearEpilogue {
    const void* bias;           /* [experts][N] or NULL                            */
    const uint16_t* residual;
    void* y;                    /* 16-bit, or fp32 where out32                     */
    uint16_t* pre;
    uint64_t ld_res, ldy, ld_pre;
    int bias_wide, act, out32;
};

struct LinearArgs {
    const uint16_t *a, *b;
    uint64_t lda, ldb;          /* elements                                        */
    uint32_t M, N, K;           /* GROUP_ROWS: M all rows; GROUP_K: K all rows     */
    /* how far the contiguous rows of a K_ROWS operand may be read (a multiple of 8) */
    uint32_t a_extent, b_extent;
    LinearEpilogue e;
    /* cut of the contraction: `splits` parts of `part_k` (a multiple of 64); with more
     * than one the sums go to part[split][M][part_ld] and a second launch joins them */
    uint32_t splits, part_k, part_ld;
    float* part;
    const int32_t* offsets;
    uint32_t experts;
    uint64_t b_stride, y_stride;   /* elements per expert: B (GROUP_ROWS), C (GROUP_K) */
    uint32_t tiles_m, tiles_n;
};

#ifdef __HIPCC__
namespace linear {

using namespace layer;

typedef int v4i_t __attribute__((ext_vector_type(4)));
typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef float v16f_t __attribute__((ext_vector_type(16)));
typedef _Float16 v8h_t __attribute__((ext_vector_type(8)));
typedef __bf16 v8b_t __attribute__((ext_vector_type(8)));

template <bool BF16> struct Half16 { typedef _Float16 T; };
template <> struct Half16<true> { typedef __bf16 T; };

/* e^x through the hardware's 2^x: relative error (|x| + 1) 2^-23 */
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

/* The complement of the error function for x >= 0, t = 1 / (1 + x/2), t exp(-x^2 + P(t)) with the
 * Chebyshev fit of Numerical Recipes (erfcc): relative error below 1.2e-7 everywhere. */
__device__ __forceinline__ float erfc_positive(float x) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.5f, x, 1.0f));
    float p = 0.17087277f;
    p = fmaf(p, t, -0.82215223f);
    p = fmaf(p, t, 1.48851587f);
    p = fmaf(p, t, -1.13520398f);
    p = fmaf(p, t, 0.27886807f);
    p = fmaf(p, t, -0.18628806f);
    p = fmaf(p, t, 0.09678418f);
    p = fmaf(p, t, 0.37409196f);
    p = fmaf(p, t, 1.00002368f);
    p = fmaf(p, t, -1.26551223f);
    return t * exp_of(fmaf(-x, x, p));
}
/* the normal distribution's integral */
__device__ __forceinline__ float normal_integral(float z) {
    const float half = 0.5f * erfc_positive(fabsf(z) * 0.70710678118654752f);
    return z < 0.0f ? half : 1.0f - half;
}
__device__ __forceinline__ float tanh_of(float z) {
    const float a = fabsf(z);
    /* below 1/4 the series to z^9 (next term below 2^-25 of z); above, no cancellation: 1 - 2 / (e^2a + 1) */
    const float s = z * z;
    float p = fmaf(s, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = fmaf(p, s, 2.0f / 15.0f);
    p = fmaf(p, s, -1.0f / 3.0f);
    const float small = fmaf(z * s, p, z);
    const float big = fmaf(-2.0f, __builtin_amdgcn_rcpf(exp_of(2.0f * a) + 1.0f), 1.0f);
    return a < 0.25f ? small : __builtin_copysignf(big, z);
}
__device__ __forceinline__ float sigmoid_of(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_of(-z)); }

__device__ __forceinline__ float act_of(float z, int act) {
    switch (act) {
    case HIP_ACT_TANH: return tanh_of(z);
    case HIP_ACT_RELU: return z < 0.0f ? 0.0f : z;              /* NaN stays NaN */
    case HIP_ACT_GELU: return z * normal_integral(z);
    case HIP_ACT_SILU: return z * sigmoid_of(z);
    default: return z;
    }
}
/* its derivative */
__device__ __forceinline__ float slope_of(float z, int act) {
    switch (act) {
    case HIP_ACT_TANH: { const float t = tanh_of(z); return fmaf(-t, t, 1.0f); }
    case HIP_ACT_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    case HIP_ACT_GELU: return fmaf(z * 0.39894228040143268f, exp_of(-0.5f * z * z), normal_integral(z));
    case HIP_ACT_SILU: { const float s = sigmoid_of(z); return s * fmaf(z, 1.0f - s, 1.0f); }
    default: return 1.0f;
    }
}

/* the group of an expert, inside 0 .. rows whatever the offsets hold */
__device__ __forceinline__ void expert_range(const int32_t* offsets, uint32_t e, uint32_t rows, uint32_t* lo, uint32_t* hi) {
    *lo = *hi = 0;
    if (rows == 0) return;                                  /* offsets may be NULL then */
    const int a = offsets[e], b = offsets[e + 1];
    const uint32_t l = a < 0 ? 0u : min((uint32_t)a, rows);
    *lo = l;
    *hi = b < 0 ? l : max(l, min((uint32_t)b, rows));
}

/* eight columns of bias row `expert` from column c on, zeros beyond N */
template <bool BF16>
__device__ __forceinline__ void load_bias(const LinearEpilogue& e, uint32_t expert, uint32_t c, uint32_t N, float (&out)[8]) {
    typedef typename Half16<BF16>::T E;
    if (!e.bias) {
#pragma unroll
        for (int i = 0; i < 8; i++) out[i] = 0.0f;
    } else if (e.bias_wide) load_row<float, float, 8>((const float*)e.bias + (uint64_t)expert * N, c, N, out);
    else load_row<E, float, 8>((const E*)e.bias + (uint64_t)expert * N, c, N, out);
}

/* z = v + bias, pre = z, y = act(z) + residual for columns c .. c + 7 of a row; y_at is the output matrix's
 * first element (its expert's, where C is one per expert) */
template <bool BF16>
__device__ __forceinline__ void finish_row8(const LinearEpilogue& e, void* y_at, uint64_t row, uint32_t c, uint32_t N,
                                            float (&v)[8], const float (&bias)[8]) {
    typedef typename Half16<BF16>::T E;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += bias[i];
    if (e.pre) store_row<E, float, 8>((E*)e.pre + row * e.ld_pre, c, N, v);
    if (e.act) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_of(v[i], e.act);
    }
    if (e.residual) {
        float r[8];
        load_row<E, float, 8>((const E*)e.residual + row * e.ld_res, c, N, r);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += r[i];
    }
    if (e.out32) store_row<float, float, 8>((float*)y_at + row * e.ldy, c, N, v);
    else store_row<E, float, 8>((E*)y_at + row * e.ldy, c, N, v);
}

}  // namespace linear
#endif
#endif
