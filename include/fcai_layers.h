/*
 * fcai_layers.h -- C ABI of the pointwise layers: the matrix product with
 * bias, activation and residual in its epilogue (tcgen05, fp32 accumulation
 * in tensor memory), layer norm, and activations whose input is kept in 8
 * bits for the backward pass, in the forms serving and training use.  They stand
 * beside the convolution layers of fcai_transforms.h for callers whose models have
 * pointwise layers too; the codecs of this library have none and do not call them.
 *
 * Tensors are rows of channels, row-major with a row stride in elements
 * (ld >= channels); channels are contiguous.  Rows are the positions of a
 * latent, the tokens of a sequence, the pixels of an NHWC activation.
 * rows = 0 is allowed everywhere: outputs over rows are left alone, sums over
 * rows are written as zeros.  Inputs and outputs do not overlap.
 *
 * Rounding: products, sums, statistics and activations are computed in fp32
 * and each output is rounded once to its type, except where a comment says
 * otherwise.
 *
 * All calls are asynchronous on `stream` of the current device and allocate
 * nothing; a call that needs scratch takes it as `workspace` (device memory,
 * 256-byte aligned, of at least the size its *_workspace function returns,
 * -1 for arguments the call would refuse), used only by that call's kernels:
 * calls that may run at the same time take different workspaces.  Status
 * codes and fcai_last_error() are those of fcai_warp_div.h.
 */
#ifndef FCAI_LAYERS_H
#define FCAI_LAYERS_H

#include <stdint.h>

#include "fcai_warp_div.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { FCAI_DTYPE_BF16 = 0, FCAI_DTYPE_F16 = 1, FCAI_DTYPE_F32 = 2 };
/* GELU is the exact form x * Phi(x); SILU is x / (1 + exp(-x)). */
enum { FCAI_ACT_NONE = 0, FCAI_ACT_RELU = 1, FCAI_ACT_GELU = 2, FCAI_ACT_SILU = 3 };
/* What a forward call keeps for its backward call.  The 8-bit forms hold, per
 * row and block of 128 channels (the last block may be shorter), one fp32
 * scale = max(amax * fl(1 / top), FLT_MIN) and codes
 * q = round(clamp(x * fl(1 / scale), +-top)): int8 (top = 127, ties to even) or
 * e4m3 (top = 448).  They read back as q * scale.  A block that holds an
 * infinity or a NaN gets the scale NaN and reads back as NaN throughout, so a
 * diverged step stays visible.  Derivatives are those of the value read back: a
 * ReLU input above 0 that rounds to 0 (below amax / 254 in int8, amax / 458752 in
 * e4m3) has the derivative 0; keep it in full where that matters.  Codes are [rows][channels] bytes, scales
 * [rows][ceil(channels / 128)] floats, both contiguous. */
enum { FCAI_KEEP_NONE = 0, FCAI_KEEP_FULL = 1, FCAI_KEEP_INT8 = 2, FCAI_KEEP_E4M3 = 3 };
#define FCAI_KEEP_BLOCK 128

/* ---- matrix product -------------------------------------------------------
 * y[rows][cout] = act(x[rows][cin] * w[cout][cin]^T + bias) + residual; bf16
 * or f16, one type for all tensors; bias and residual may be NULL.  `keep` says
 * what of p = x * w^T + bias, the activation's input, stays for the backward
 * pass: NONE; FULL, p rounded to the type in pre; INT8 or E4M3, p (before any
 * rounding) as codes and scales.  Addresses and strides need only the elements'
 * alignment; 16-byte aligned addresses and strides (8 elements) are read
 * without a copy.  With an 8-bit keep, more than 32 rows and cout a multiple of
 * 8, the addresses and strides of y, bias and residual, and codes, are 16-byte
 * aligned.  With an 8-bit keep and cout no multiple of 16 the workspace holds p
 * as fp32 (below 6 Mi values) or the codes in padded rows; it also holds p as
 * fp32 up to 32 rows, and any product's partial sums where cin is split. */
enum { FCAI_LINEAR_FORWARD = 0, FCAI_LINEAR_BACKWARD_INPUT = 1, FCAI_LINEAR_BACKWARD_WEIGHT = 2 };
/* `repack`: bits set for matrices of the call that are not 16-byte aligned in
 * address and row stride: 1 the first operand (x; dp; dp), 2 the second (w; w;
 * x), 4 the output (y; dx; dw), 8 the residual, and 16 for a bias whose address
 * is not, or whose length is no multiple of 8.  `keep`: the forward call's (0 for
 * the others). */
int64_t fcai_linear_workspace(int32_t op, int64_t rows, int32_t cin, int32_t cout, int32_t repack, int32_t keep);
int fcai_linear_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *bias,
                        const void *residual, int64_t ldr, void *y, int64_t ldy, void *pre, int64_t ldpre,
                        void *codes, float *scales, int64_t rows, int32_t cin, int32_t cout, int32_t dtype, int32_t act,
                        int32_t keep, void *workspace, int64_t workspace_bytes, fcai_stream_t stream);
/* The kernels' waits are bounded.  One that runs out (a bug, never expected)
 * ends its product early and sets its device's word (host memory; this returns
 * the current device's, NULL without a device).  The next call that launches a
 * product on that device clears the word and returns FCAI_ERR_CUDA instead of
 * running.  Replays of a captured graph make no such call, and the last product
 * has none after it: read the word, and clear it, after a synchronise. */
int32_t *fcai_linear_error_word(void);
/* dx[rows][cin] = dp[rows][cout] * w[cout][cin] */
int fcai_linear_backward_input(const void *dp, int64_t lddp, const void *w, int64_t ldw, void *dx, int64_t lddx,
                               int64_t rows, int32_t cin, int32_t cout, int32_t dtype, void *workspace,
                               int64_t workspace_bytes, fcai_stream_t stream);
/* dw[cout][cin] = dp[rows][cout]^T * x[rows][cin] */
int fcai_linear_backward_weight(const void *dp, int64_t lddp, const void *x, int64_t ldx, void *dw, int64_t lddw,
                                int64_t rows, int32_t cin, int32_t cout, int32_t dtype, void *workspace,
                                int64_t workspace_bytes, fcai_stream_t stream);

/* ---- activations and 8-bit checkpoints --------------------------------------
 * y = act(x) (skipped when y is NULL) and, for an 8-bit keep, x's codes and
 * scales.  bf16, f16 or f32. */
int fcai_activation_forward(const void *x, int64_t ldx, void *y, int64_t ldy, void *codes, float *scales,
                            int64_t rows, int32_t channels, int32_t dtype, int32_t act, int32_t keep,
                            fcai_stream_t stream);
/* dx = dy * act'(x), x from the tensor itself (keep FULL, x/ldx) or from its
 * codes and scales.  bias_grad (channels elements of the type, or NULL)
 * receives the column sums of the unrounded dx; dx may be NULL then.  With
 * act NONE nothing of x is read. */
int64_t fcai_activation_workspace(int64_t rows, int32_t channels);
int fcai_activation_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *codes,
                             const float *scales, void *dx, int64_t lddx, void *bias_grad, int64_t rows,
                             int32_t channels, int32_t dtype, int32_t act, int32_t keep, void *workspace,
                             int64_t workspace_bytes, fcai_stream_t stream);
/* The values an 8-bit checkpoint stands for, rounded to `dtype`. */
int fcai_checkpoint_load(const void *codes, const float *scales, void *out, int64_t ldo, int64_t rows,
                         int32_t channels, int32_t dtype, int32_t keep, fcai_stream_t stream);

/* ---- layer norm -------------------------------------------------------------
 * y = (x - mean) * rstd * weight + bias over the channels of each row, the
 * variance from the centred values, rstd = 1 / sqrt(var + eps).  weight and
 * bias (both may be NULL: 1 and 0) have type wdtype: x's type or f32.  mean
 * and rstd (rows floats each, or both NULL) and, for an 8-bit keep, x's codes
 * and scales are written for the backward call. */
int fcai_layer_norm_forward(const void *x, int64_t ldx, const void *weight, const void *bias, int32_t wdtype,
                            void *y, int64_t ldy, float *mean, float *rstd, void *codes, float *scales, int64_t rows,
                            int32_t channels, float eps, int32_t dtype, int32_t keep, fcai_stream_t stream);
/* With t = dy * weight and xhat = (x - mean) * rstd:
 * dx = rstd * (t - mean(t) - xhat * mean(t * xhat)), dweight = sum over rows of
 * dy * xhat, dbias = sum of dy (both of wdtype, either may be NULL). */
int64_t fcai_layer_norm_workspace(int64_t rows, int32_t channels);
int fcai_layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, const void *codes,
                             const float *scales, const float *mean, const float *rstd, const void *weight,
                             int32_t wdtype, void *dx, int64_t lddx, void *dweight, void *dbias, int64_t rows,
                             int32_t channels, int32_t dtype, int32_t keep, void *workspace, int64_t workspace_bytes,
                             fcai_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FCAI_LAYERS_H */
