/* bptbias — a learned bias of attention scores by buckets (libbptbias, gfx950): every edge has a bucket, every bucket and head a scalar.
 *
 * Device pointers, sizes, a hipStream_t; the return value is 0, a negative bpt_status (bptattn.h: nothing was launched) or a
 * positive hipError_t.  Nothing is allocated or synchronised; everything is deterministic.  A bucket outside of 0 .. n_buckets - 1 stands for
 * no bias: it adds 0 and has no gradient.
 */
#ifndef BPTBIAS_H
#define BPTBIAS_H

#include <stdint.h>

#include "bptscore.h"

#ifdef __cplusplus
extern "C" {
#endif

/* bias[e][head] = table[buckets[e]][head] * factor; table (n_buckets, h) of dtype, buckets (n_edges), bias (n_edges, h) of out_dtype: dtype, or BPT_F32
 * where that is BPT_BF16.  spare_row: bias has a row more, which becomes 0 (what bpt_attention_forward's bias is). */
int bpt_bucket_bias_forward(const void *table, const int64_t *buckets, void *bias, int64_t n_edges, int64_t n_buckets, int h, double factor,
                            int spare_row, int dtype, int out_dtype, void *stream);

/* dtable[b][head] = factor * the sum of ds[e][head] over the edges of bucket b; ds (n_edges, h) of ds_dtype, dtable (n_buckets, h) of dtype. */
int64_t bpt_bucket_bias_backward_workspace_bytes(int64_t n_edges, int64_t n_buckets, int h, int dtype);
int bpt_bucket_bias_backward(const void *ds, const int64_t *buckets, void *dtable, void *workspace, int64_t workspace_bytes, int64_t n_edges,
                             int64_t n_buckets, int h, double factor, int dtype, int ds_dtype, void *stream);

/* The fused pass of bptscore.h with u = scale (q[dst].k[src]) + table[bucket][head], capped and lowered by distance or not (score as there; all of it 0: neither).
 * Heads of 64 columns, h = 8 or 16 of them, float32 also 4; up to 255 buckets.  Plans as there, with grp_eids on either side.  scale is not 0.  In bfloat16 delta comes from
 * the pairs.  Values of -BPT_HIDES and below in table, -infinity among them, hide a bucket's edges (with a cap: their scores are -cap); a row with nothing left is 0. */
#define BPT_MOST_BUCKETS 255
#define BPT_HIDES 524288.0f

/* What the passes of a call take: the heads' tables and the bucket of every place of the plans, written to `prepared` (on 16 bytes).  plan_out may be NULL where no
 * backward follows.  table (n_buckets, heads) of dtype, heads <= h (those behind have no bias), buckets (n_edges). */
int64_t bpt_bucket_prepare_bytes(const bpt_plan *plan_in, const bpt_plan *plan_out, int h);
int bpt_bucket_prepare(const bpt_plan *plan_in, const bpt_plan *plan_out, const void *table, const int64_t *buckets, int64_t n_buckets, int heads, int h,
                       float scale, int dtype, void *prepared, void *stream);

/* The workspace is that of bpt_score_forward. */
int bpt_bucket_attention_forward(const bpt_plan *plan_in, const bpt_score *score, const void *prepared, const void *q, const void *k, const void *v, void *o,
                                 float *lse, void *workspace, int64_t workspace_bytes, float scale, float dropout_p, uint64_t dropout_seed, int h, int dtype,
                                 void *stream);

/* dtable (n_buckets, heads) of dtype or NULL; the rest as bpt_score_backward. */
int64_t bpt_bucket_attention_backward_workspace_bytes(const bpt_plan *plan_in, const bpt_plan *plan_out, int64_t n_buckets, int heads, int h, int dtype);
int bpt_bucket_attention_backward(const bpt_plan *plan_in, const bpt_plan *plan_out, const bpt_score *score, const void *prepared, const void *q, const void *k,
                                  const void *v, const void *o, const void *d_o, const float *lse, void *dq, void *dk, void *dv, void *dtable,
                                  float *dslopes, void *workspace, int64_t workspace_bytes, int64_t n_buckets, int heads, float scale, float dropout_p,
                                  uint64_t dropout_seed, int h, int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif
