/*
 * Layers of a feed-forward block as models train and serve it: layer norm, the
 * linear layer with bias, activation and residual in the product's epilogue, and
 * the same layer held once per expert for rows that are grouped by expert; each
 * with its gradients. They stand beside the products of gpu_hip_tiers.h
 * (hip_hgemm_16, hip_bias_act_f64, the batched entry points) and have no
 * counterpart in the reference, whose layers run on the host.
 *
 * Conventions: plain C, device pointers, arguments in a struct that the callee
 * only reads, `stream` is a hipStream_t passed as void* (NULL = the null stream).
 * Return 0 on success, -1 on a bad argument, an unsupported size or a launch
 * failure, -2 when the workspace is missing or too small; with
 * ESHKOL_GPU_VERBOSE=1 a refusal says why on stderr. A refused call has queued
 * nothing. Zero a struct before filling it: fields added later mean "no" as 0.
 *
 * Element types are the runtime's dtype codes: 0 f64, 1 f32, 2 f16, 3 bf16.
 * Matrices are row-major with a pitch in elements (ld...) of at least a row's
 * length; rows and pointers need the alignment of an element and no more
 * (16-byte aligned rows are faster). A pitch may be given as 0: the row's length.
 *
 * Memory. The calls allocate nothing, synchronise nothing and keep nothing of a
 * call: they touch only the memory they are given, so they may be called from any
 * thread, on any stream, and be captured into a graph. (What the process does keep
 * is which kernels have been given their LDS on which device, under a lock held for
 * a look at that list; a kernel's first call registers it.) Those
 * that need scratch take it from the caller: fill in everything else, ask the
 * *_workspace function (host arithmetic only; -1 where the call itself would
 * refuse the arguments), and pass at least so many bytes, 16-byte aligned. Its
 * contents mean nothing before or after the call. Two calls that can run at the
 * same time, and two captured graphs that can, need a workspace each. Pointers must be
 * usable on the stream's device, which need not be the current one.
 *
 * Results do not depend on timing: every sum is taken in an order that the call
 * fixes, by its sizes and types, the alignment of its pointers and pitches, which
 * outputs it asks for, and the device's CU count. The same call gives the same bits;
 * one that asks for other outputs too, or has the same values at another alignment,
 * may add in another order and round differently. Sums, means and deviations are
 * held in fp32 (f64 tensors: f64), and an output is rounded once; fp32 results below
 * 2^-119 may come out as 0 (the hardware's exponential has no subnormal results).
 */
#ifndef ESHKOL_GPU_HIP_LAYERS_H
#define ESHKOL_GPU_HIP_LAYERS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* act: the activations of the linear layer and of the experts */
enum {
    HIP_ACT_NONE = 0,
    HIP_ACT_TANH = 1,       /* the code hip_bias_act_f64 has for it */
    HIP_ACT_RELU = 2,       /* derivative 0 at 0 */
    HIP_ACT_GELU = 3,       /* z Phi(z), Phi the normal distribution's integral (no tanh form) */
    HIP_ACT_SILU = 4        /* z / (1 + e^-z) */
};                          /* at an infinity: the limit (gelu and silu 0 at -infinity); NaN stays NaN */

/* ---- layer norm --------------------------------------------------------------
 * y = (x - mean) rstd gamma + beta for every row of `cols` elements,
 * mean = sum x / cols, rstd = 1 / sqrt(sum (x - mean)^2 / cols + epsilon).
 * dtype 0 .. 3; gamma and beta are of param_dtype: dtype itself, or 1 beside a
 * 16-bit dtype. mean and rstd (one per row, fp32; f64 for dtype 0) are what the
 * backward pass takes; NULL where nothing follows. y may be x (with its pitch).
 * rows may be 0. cols at most 2^24, rows at most 2^40. */
typedef struct {
    const void* x;          /* [rows][cols]                                        */
    const void* gamma;      /* [cols], NULL: ones                                  */
    const void* beta;       /* [cols], NULL: zeros                                 */
    void* y;                /* [rows][cols]                                        */
    void* mean;             /* [rows] or NULL                                      */
    void* rstd;             /* [rows] or NULL                                      */
    uint64_t rows, cols;
    uint64_t ldx, ldy;
    double epsilon;         /* finite, >= 0                                        */
    int32_t dtype, param_dtype;
} HipLayerNormArgs;
int hip_layernorm(const HipLayerNormArgs* args, void* stream);

/* Its gradients, with h = (x - mean) rstd and t = grad_y gamma:
 *   grad_x     = rstd (t - sum t / cols - h sum (t h) / cols) [+ grad_residual]
 *   grad_gamma = sum over rows of grad_y h,   grad_beta = sum over rows of grad_y
 * grad_residual is the gradient that reaches x around the layer (a residual
 * block), NULL for none. grad_gamma and grad_beta are fp32 (f64 for dtype 0) and
 * overwritten; zeros for rows == 0. Any of the three outputs may be NULL, not all.
 * grad_x may be grad_y, x or grad_residual (with its pitch). */
typedef struct {
    const void* grad_y;         /* [rows][cols]                                    */
    const void* x;              /* [rows][cols]                                    */
    const void* gamma;          /* [cols], NULL: ones                              */
    const void* mean;           /* [rows], of the forward pass                     */
    const void* rstd;           /* [rows]                                          */
    const void* grad_residual;  /* [rows][cols] or NULL                            */
    void* grad_x;               /* [rows][cols] or NULL                            */
    void* grad_gamma;           /* [cols] or NULL                                  */
    void* grad_beta;            /* [cols] or NULL                                  */
    uint64_t rows, cols;
    uint64_t ld_grad_y, ldx, ld_grad_residual, ld_grad_x;
    int32_t dtype, param_dtype;
    void* workspace;
    uint64_t workspace_bytes;
} HipLayerNormBackwardArgs;
int64_t hip_layernorm_backward_workspace(const HipLayerNormBackwardArgs* args);
int hip_layernorm_backward(const HipLayerNormBackwardArgs* args, void* stream);

/* ---- linear layer ------------------------------------------------------------
 * z = x W + bias,  y = act(z) + residual,  pre = z
 * on the matrix cores, dtype 2 (f16) or 3 (bf16), sums and epilogue in fp32, y and
 * pre rounded once each (act is applied to the unrounded z). W is [K][N], or
 * [N][K] with trans_w != 0. bias is of param_dtype (dtype or 1). pre is what the
 * backward pass of an activation takes; NULL where nothing follows. y may be
 * residual (with its pitch); no other output may overlap an input. M may be 0;
 * M below 2^31, K and N at most 2^22. */
typedef struct {
    const void* x;          /* [M][K]                                              */
    const void* w;          /* [K][N], trans_w: [N][K]                             */
    const void* bias;       /* [N] or NULL                                         */
    const void* residual;   /* [M][N] or NULL                                      */
    void* y;                /* [M][N]                                              */
    void* pre;              /* [M][N] or NULL                                      */
    uint64_t M, K, N;
    uint64_t ldx, ldw, ld_residual, ldy, ld_pre;
    int32_t dtype, param_dtype, act, trans_w;
    void* workspace;
    uint64_t workspace_bytes;
} HipLinearArgs;
int64_t hip_linear_16_workspace(const HipLinearArgs* args);
int hip_linear_16(const HipLinearArgs* args, void* stream);

/* Its gradients, with dz = grad_y act'(pre):
 *   grad_x = dz W^T,   grad_w = x^T dz (of W's shape),   grad_bias = sum over rows of dz
 * pre is read only for act != 0. dz is rounded to dtype before it enters the two
 * products (the operand type of the matrix cores); grad_bias, fp32, sums it
 * unrounded. grad_w is of grad_w_dtype: dtype, or 1. The gradient of the residual
 * is grad_y itself. Any output may be NULL, not all; M may be 0 (grad_w and
 * grad_bias are then zeros). No output may overlap an input. */
typedef struct {
    const void* grad_y;     /* [M][N]                                              */
    const void* pre;        /* [M][N], or NULL for act 0                           */
    const void* x;          /* [M][K], may be NULL where grad_w is                 */
    const void* w;          /* may be NULL where grad_x is                         */
    void* grad_x;           /* [M][K] or NULL                                      */
    void* grad_w;           /* [K][N] (trans_w: [N][K]) or NULL                    */
    void* grad_bias;        /* [N] fp32 or NULL                                    */
    uint64_t M, K, N;
    uint64_t ld_grad_y, ld_pre, ldx, ldw, ld_grad_x, ld_grad_w;
    int32_t dtype, grad_w_dtype, act, trans_w;
    void* workspace;
    uint64_t workspace_bytes;
} HipLinearBackwardArgs;
int64_t hip_linear_backward_16_workspace(const HipLinearBackwardArgs* args);
int hip_linear_backward_16(const HipLinearBackwardArgs* args, void* stream);

/* ---- the linear layer by expert -------------------------------------------------
 * The rows of x are grouped by expert: those of expert e are offsets[e] ..
 * offsets[e+1] - 1, and they are multiplied by W_e = w + e w_stride, with bias row
 * e. offsets, experts + 1 of them in device memory, are read on the device (a
 * router's output needs no trip to the host), ascending from at least 0 to at
 * most rows; an expert may have no rows. Rows before offsets[0] and behind
 * offsets[experts] belong to no expert: their outputs are left as they were.
 * (Offsets that do not ascend, or lie outside 0 .. rows, give meaningless results, but no access
 * outside the tensors.) experts at most 4096, rows below 2^31; otherwise as
 * hip_linear_16, without a residual. w_stride 0: the experts' matrices back to back. */
typedef struct {
    const void* x;          /* [rows][K]                                           */
    const void* w;          /* [experts][K][N], trans_w: [experts][N][K]           */
    const void* bias;       /* [experts][N] or NULL                                */
    const int32_t* offsets; /* [experts + 1]                                       */
    void* y;                /* [rows][N]                                           */
    void* pre;              /* [rows][N] or NULL                                   */
    uint64_t rows, experts, K, N;
    uint64_t ldx, ldw, w_stride, ldy, ld_pre;
    int32_t dtype, param_dtype, act, trans_w;
    void* workspace;
    uint64_t workspace_bytes;
} HipExpertsArgs;
int64_t hip_experts_16_workspace(const HipExpertsArgs* args);
int hip_experts_16(const HipExpertsArgs* args, void* stream);

/* Its gradients, as hip_linear_backward_16 for every expert: grad_w and grad_bias
 * of an expert without rows are zeros; rows of grad_x that belong to no expert are
 * left as they were. */
typedef struct {
    const void* grad_y;     /* [rows][N]                                           */
    const void* pre;        /* [rows][N], or NULL for act 0                        */
    const void* x;          /* [rows][K], may be NULL where grad_w is              */
    const void* w;          /* may be NULL where grad_x is                         */
    const int32_t* offsets; /* [experts + 1]                                       */
    void* grad_x;           /* [rows][K] or NULL                                   */
    void* grad_w;           /* of w's shape, or NULL                               */
    void* grad_bias;        /* [experts][N] fp32 or NULL                           */
    uint64_t rows, experts, K, N;
    uint64_t ld_grad_y, ld_pre, ldx, ldw, w_stride, ld_grad_x, ld_grad_w, grad_w_stride;
    int32_t dtype, grad_w_dtype, act, trans_w;
    void* workspace;
    uint64_t workspace_bytes;
} HipExpertsBackwardArgs;
int64_t hip_experts_backward_16_workspace(const HipExpertsBackwardArgs* args);
int hip_experts_backward_16(const HipExpertsBackwardArgs* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif
