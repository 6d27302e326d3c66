/* bptscore — attention over a graph whose scores are capped and / or fall with distance (libbptscore, gfx950).
 *
 * The fused pass of bptattn.h (bpt_attention_forward / _backward) with, for an edge and head and u = (q[dst].k[src] + bias) scale,
 *   s = cap tanh(u / cap)   (s = u where cap is 0)   - slopes[head] |pos_q[dst] - pos_k[src]|   (where slopes is given)
 * in place of u.  Heads of 64 columns; float32 with 4, 8 or 16 of them, bfloat16 with 8 or 16; without a bias also heads of 4 to 64 columns as
 * they are (bfloat16: of an even number of columns; rows start on 4 bytes), `heads` of them, computed as h = 4, 8 or 16, which is what lse (n, h),
 * the workspace and dropout's hash count.  Plans carry groups of 16 rows (tiles), the source side's the pair numbers of the destination side's;
 * grp_eids where there is dropout or a bias.  A forward on a plan without groups walks single rows (heads of 64 columns, no dropout, no bias): few
 * rows of many edges.  Conventions, status codes, plans, bias, ds_out, dropout and lse are those of bptattn.h (bias by edge id: bias_by_pair is
 * refused; a row with a NaN score is NaN, and so is its lse; scores may lie as low as -2 * 10^38, held in 32 bits: with m the largest of a row's, they and
 * its lse are off by a few 2^-24 |m|, an exponent's error in its probabilities).  Deterministic; nothing is allocated.
 */
#ifndef BPTSCORE_H
#define BPTSCORE_H

#include <stdint.h>

#include "bptattn.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    float cap;                        /* 0: not capped; otherwise between 10^-10 and 10^10 and at least |scale| / 10^4, with |scale| <= 10^6 */
    const float *slopes;              /* (heads) float32, or NULL: no distance */
    const float *pos_q, *pos_k;       /* float32 positions of the query rows and of the key rows, with slopes */
} bpt_score;

int64_t bpt_score_forward_workspace_bytes(const bpt_plan *plan_in, int h);
int64_t bpt_score_backward_workspace_bytes(const bpt_plan *plan_in, const bpt_plan *plan_out, int h, int dtype, int has_bias);

int bpt_score_forward(const bpt_plan *plan_in, const bpt_score *score, const void *q, const void *k, const void *v, const float *bias, void *o, float *lse,
                      void *workspace, int64_t workspace_bytes, float scale, float dropout_p, uint64_t dropout_seed, int heads, int d, int h, int dtype,
                      void *stream);

/* ds_out goes with bias; dslopes (heads) float32 or NULL: dL/dslopes = -sum over the edges of dL/ds |pos_q[dst] - pos_k[src]|. */
int bpt_score_backward(const bpt_plan *plan_in, const bpt_plan *plan_out, const bpt_score *score, const void *q, const void *k, const void *v,
                       const float *bias, const void *o, const void *d_o, const float *lse, void *dq, void *dk, void *dv, float *ds_out, float *dslopes,
                       void *workspace, int64_t workspace_bytes, float scale, float dropout_p, uint64_t dropout_seed, int heads, int d, int h, int dtype,
                      void *stream);

#ifdef __cplusplus
}
#endif
#endif
