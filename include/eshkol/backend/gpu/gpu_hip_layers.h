/*
 * Layers of a feed-forward block as models train and serve it: layer norm with its
 * gradients. They stand beside the products and streaming kernels of
 * gpu_hip_tiers.h.
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
 * Memory. The calls allocate nothing, take no lock, keep nothing between calls
 * and synchronise nothing: they touch only the memory they are given, so they may
 * be called from any thread, on any stream, and be captured into a graph. Those
 * that need scratch take it from the caller: fill in everything else, ask the
 * *_workspace function (host arithmetic only; -1 where the call itself would
 * refuse the arguments), and pass at least so many bytes, 16-byte aligned. Its
 * contents mean nothing before or after the call. Two calls that can run at the
 * same time, and two captured graphs that can, need a workspace each. Pointers must be
 * usable on the stream's device, which need not be the current one.
 *
 * Results do not depend on timing: every sum is taken in an order that the sizes
 * and the device's CU count fix. Sums, means and deviations are held in fp32 (f64
 * tensors: f64), and an output is rounded once.
 */
#ifndef ESHKOL_GPU_HIP_LAYERS_H
#define ESHKOL_GPU_HIP_LAYERS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

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

#ifdef __cplusplus
}
#endif
#endif
