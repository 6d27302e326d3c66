/* bptbias — a learned bias of attention scores by buckets (libbptbias, gfx950): every edge has a bucket, every bucket and head a scalar.
 *
 * Device pointers, sizes, a hipStream_t; the return value is 0, a negative bpt_status (bptattn.h: nothing was launched) or a
 * positive hipError_t.  Nothing is allocated or synchronised; everything is deterministic.  A bucket outside of 0 .. n_buckets - 1 stands for
 * no bias: it adds 0 and has no gradient.
 */
#ifndef BPTBIAS_H
#define BPTBIAS_H

#include <stdint.h>

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

/* The same in the order of a tile plan's pairs (bias_by_pair of bptattn.h).  eid_of_pair (n_edges) int32: the edge of every pair number; codes (n_edges)
 * uint16: the buckets of the pairs, 65535 where there is none; bias (h, n_edges) float32.  n_buckets <= 65535. */
int bpt_bucket_pairs_forward(const void *table, const int64_t *buckets, const int32_t *eid_of_pair, uint16_t *codes, float *bias, int64_t n_edges,
                             int64_t n_buckets, int h, double factor, int dtype, void *stream);

/* ds (h, n_edges) float32; the workspace is that of bpt_bucket_bias_backward. */
int bpt_bucket_pairs_backward(const float *ds, const uint16_t *codes, void *dtable, void *workspace, int64_t workspace_bytes, int64_t n_edges,
                              int64_t n_buckets, int h, double factor, int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif
