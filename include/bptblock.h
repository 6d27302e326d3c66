/* bptblock — the operators of a transformer block around its attention (libbptblock, gfx950).
 *
 * Device pointers, sizes, a hipStream_t; the return value is 0, a negative bpt_status (bptattn.h: nothing was launched) or a
 * positive hipError_t.  Nothing is allocated or synchronised; everything is deterministic.  dtype: BPT_F32, BPT_F64 or BPT_BF16 (relu8:
 * BPT_F32 or BPT_BF16).  Tensors are contiguous; any alignment of the element's size is accepted.
 */
#ifndef BPTBLOCK_H
#define BPTBLOCK_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Layer norm of a sum over the last axis, y = (z - mean) rstd weight + bias with z = x + residual, (rows, cols) each.
 * residual, weight and bias may be NULL (none; ones; zeros).  stats: NULL, or (rows, 2) of the accumulation type (float; double for
 * BPT_F64): mean and rstd = 1 / sqrt(variance + eps), which the backward reads. */
int bpt_add_norm_forward(const void *x, const void *residual, const void *weight, const void *bias, void *y, void *stats, int64_t rows,
                         int64_t cols, double eps, int dtype, void *stream);

/* dz = dL/dz (the gradient of x and of residual), and where not NULL dweight = sum over the rows of dy xhat, dbias = sum of dy; for
 * either the workspace is needed.  dz may be NULL too, and stats where neither dz nor dweight is wanted. */
int64_t bpt_add_norm_workspace_bytes(int64_t rows, int64_t cols, int dtype);
int bpt_add_norm_backward(const void *x, const void *residual, const void *weight, const void *stats, const void *dy, void *dz, void *dweight,
                          void *dbias, void *workspace, int64_t workspace_bytes, int64_t rows, int64_t cols, int dtype, void *stream);

/* Activations that share a step. */
#define BPT_RELU8_BLOCK 64
/* exps value of a block with an activation that is infinite or NaN: its codes stand for NaN. */
#define BPT_RELU8_NAN 127

/* y = relu(a), or with dropout relu(a) / (1 - p) where a hash of (seed, index) keeps the element and 0 elsewhere, n elements, and y in
 * 8 bits: every 64 neighbouring elements share a step 2^e, e (exps, ceil(n / 64)) the smallest exponent >= -126 with max(y) <= 255 2^e, and
 * codes = y / 2^e rounded to the nearest (ties to even), 1 at least where y > 0.  y may be NULL.  n < 2^32 with dropout. */
int bpt_relu8_forward(const void *a, void *y, uint8_t *codes, int8_t *exps, int64_t n, float dropout_p, uint64_t dropout_seed, int dtype,
                      void *stream);
/* da = dy / (1 - p) where the code is not 0, else 0; y8 = code 2^e, what the codes stand for.  Either may be NULL; da may be dy. */
int bpt_relu8_backward(const void *dy, const uint8_t *codes, const int8_t *exps, void *da, void *y8, int64_t n, float dropout_p, int dtype,
                       void *stream);

#ifdef __cplusplus
}
#endif
#endif
