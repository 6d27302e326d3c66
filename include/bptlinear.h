/* bptlinear — matrix products with an epilogue, dropout from a counter-based generator (libbptlinear, gfx950).
 *
 * Device pointers, sizes, a hipStream_t; the return value is 0, a negative bpt_status (bptattn.h: nothing was launched) or a
 * positive hipError_t.  Nothing is allocated or synchronised; everything is deterministic.  dtype: BPT_F32 or BPT_BF16.  Tensors are
 * contiguous; any alignment of the element's size is accepted, workspaces start on 16 bytes.  Sums are held in 32 bits.
 *
 * Dropout: element i (its place in memory) takes word i % 4 of Philox-4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011) of the
 * counter (i / 4, 0) under the key seed.  It becomes 0 where the word is below the whole part of dropout_p 2^32 (1 where that
 * is less, 2^32 - 1 at most) and is divided by 1 - dropout_p elsewhere.
 */
#ifndef BPTLINEAR_H
#define BPTLINEAR_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { BPT_ACT_NONE = 0, BPT_ACT_RELU = 1, BPT_ACT_GELU = 2 } bpt_act;      /* GELU: a (1 + erf(a / sqrt 2)) / 2 */

/* y = residual + dropout(act(a)), a = x weight^T + bias; x (rows, inner), weight (outer, inner), bias (outer) or NULL, residual (rows, outer) or NULL.
 * kept: NULL, or (rows, outer), which receives a in dtype for the backward.  inner >= 1. */
int64_t bpt_linear_forward_workspace_bytes(int64_t rows, int64_t inner, int64_t outer, int dtype);
int bpt_linear_forward(const void *x, const void *weight, const void *bias, const void *residual, void *y, void *kept, void *workspace,
                       int64_t workspace_bytes, int64_t rows, int64_t inner, int64_t outer, int act, double dropout_p, uint64_t seed, int dtype,
                       void *stream);

/* g = dy act'(a) where dropout keeps the element, 0 elsewhere, (rows, outer), and where dbias is not NULL its sums over the rows divided by 1 - dropout_p; the workspace
 * is for these.  g is not divided: the two products below take 1 / (1 - dropout_p) as scale.  g may be NULL, and may be dy.
 * kept: the forward's kept tensor, or, with BPT_ACT_RELU and kept_is_result, its y (which had no residual); not read without an activation. */
int64_t bpt_linear_grad_workspace_bytes(int64_t rows, int64_t outer, int dtype);
int bpt_linear_grad(const void *dy, const void *kept, int kept_is_result, void *g, void *dbias, void *workspace, int64_t workspace_bytes,
                    int64_t rows, int64_t outer, int act, double dropout_p, uint64_t seed, int dtype, void *stream);

/* dx = scale g weight, (rows, inner). */
int64_t bpt_linear_input_grad_workspace_bytes(int64_t rows, int64_t inner, int64_t outer, int dtype);
int bpt_linear_input_grad(const void *g, const void *weight, void *dx, void *workspace, int64_t workspace_bytes, int64_t rows, int64_t inner,
                          int64_t outer, double scale, int dtype, void *stream);

/* dweight = scale g^T x, (outer, inner). */
int64_t bpt_linear_weight_grad_workspace_bytes(int64_t rows, int64_t inner, int64_t outer, int dtype);
int bpt_linear_weight_grad(const void *g, const void *x, void *dweight, void *workspace, int64_t workspace_bytes, int64_t rows, int64_t inner,
                           int64_t outer, double scale, int dtype, void *stream);

/* y = residual + dropout(x), n elements (at most 2^36 - 4096 in float32, 2^37 - 8192 in bfloat16); residual may be NULL.  y may be x or residual.  The gradient of x is the same call on dy without a residual. */
int bpt_dropout(const void *x, const void *residual, void *y, int64_t n, double dropout_p, uint64_t seed, int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif
