// libbptscore: C ABI (include/bptscore.h) of the fused attention with capped scores and distance.
#include "bptmod.h"

extern "C" {

int64_t bpt_score_forward_workspace_bytes(const bpt_plan *plan_in, int h) {
    return plan_in && h > 0 ? round16(plan_in->n_slots * ((int64_t)h * 64 + 2 * h) * 4) : -1;
}

int64_t bpt_score_backward_workspace_bytes(const bpt_plan *plan_in, const bpt_plan *plan_out, int h, int dtype, int has_bias) {
    if (!plan_in || !plan_out || h < 1 || (dtype != BPT_F32 && dtype != BPT_BF16)) return -1;
    return scratch_bytes(plan_in, plan_out, h, dtype, has_bias != 0) + slope_bytes(plan_in, h) + split_bytes(plan_in, h, dtype == BPT_BF16 && !has_bias) +
           round16((plan_in->n_slots + 2 * plan_out->n_slots) * (int64_t)h * 64 * 4);
}

int bpt_score_forward(const bpt_plan *plan_in, const bpt_score *score, const void *q, const void *k, const void *v, const float *bias, void *o, float *lse,
                      void *workspace, int64_t workspace_bytes, float scale, float dropout_p, uint64_t dropout_seed, int heads, int d, int h, int dtype,
                      void *stream) {
    Narrow nw;
    const int st = check_score(plan_in, score, heads, d, h, dtype, scale, dropout_p, bias, nw, true);
    if (st != BPT_OK) return st;
    if (plan_in->n_rows == 0) return BPT_OK;
    if (!q || !k || !v || !o || !lse) return BPT_ERR_NULL;
    if (!aligned16(workspace) || (nw.heads == 0 ? !on16({q, k, v, o}) : !on4({q, k, v, o}))) return BPT_ERR_UNSUPPORTED;
    const int64_t need = bpt_score_forward_workspace_bytes(plan_in, h);
    if (need > 0 && (!workspace || workspace_bytes < need)) return BPT_ERR_WORKSPACE;
    const Dropout drop = make_dropout(dropout_p, dropout_seed);
    if (nw.heads > 0)
        return dtype == BPT_F32 ? run_forward_narrow<float>(plan_in, score, q, k, v, o, lse, workspace, scale, drop, nw, (hipStream_t)stream)
                                : run_forward_narrow<bf16_t>(plan_in, score, q, k, v, o, lse, workspace, scale, drop, nw, (hipStream_t)stream);
    DISPATCH((run_forward<T, H>(plan_in, score, q, k, v, bias, o, lse, workspace, scale, drop, (hipStream_t)stream)))
}

int bpt_score_backward(const bpt_plan *plan_in, const bpt_plan *plan_out, const bpt_score *score, const void *q, const void *k, const void *v,
                       const float *bias, const void *o, const void *d_o, const float *lse, void *dq, void *dk, void *dv, float *ds_out, float *dslopes,
                       void *workspace, int64_t workspace_bytes, float scale, float dropout_p, uint64_t dropout_seed, int heads, int d, int h, int dtype,
                      void *stream) {
    Narrow nw;
    int st = check_score(plan_in, score, heads, d, h, dtype, scale, dropout_p, bias, nw, false);
    if (st != BPT_OK) return st;
    st = check_plan(plan_out, true);
    if (st != BPT_OK) return st;
    if (plan_in->n_edges != plan_out->n_edges) return BPT_ERR_PLAN;
    if (plan_in->n_groups == 0 || !has_tiles(plan_out, h, 64, dtype == BPT_BF16 ? 2 : 4) || !plan_out->grp_pairs) return BPT_ERR_UNSUPPORTED;
    if ((bias != nullptr) != (ds_out != nullptr) || (dslopes && !score->slopes)) return BPT_ERR_NULL;
    if (dropout_p > 0.f && dtype == BPT_BF16 && !bias && !plan_out->grp_eids) return BPT_ERR_PLAN;
    if (!q || !k || !v || !o || !d_o || !lse || !dq || !dk || !dv) return BPT_ERR_NULL;
    if (!aligned16(workspace) || (nw.heads == 0 ? !on16({q, k, v, o, d_o, dq, dk, dv}) : !on4({q, k, v, o, d_o, dq, dk, dv}))) return BPT_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < bpt_score_backward_workspace_bytes(plan_in, plan_out, h, dtype, bias != nullptr)) return BPT_ERR_WORKSPACE;
    const Dropout drop = make_dropout(dropout_p, dropout_seed);
    if (nw.heads > 0)
        return dtype == BPT_F32 ? run_backward_narrow<float>(plan_in, plan_out, score, q, k, v, o, d_o, lse, dq, dk, dv, dslopes, workspace, scale, drop, nw, (hipStream_t)stream)
                                : run_backward_narrow<bf16_t>(plan_in, plan_out, score, q, k, v, o, d_o, lse, dq, dk, dv, dslopes, workspace, scale, drop, nw, (hipStream_t)stream);
    DISPATCH((run_backward<T, H>(plan_in, plan_out, score, q, k, v, bias, o, d_o, lse, dq, dk, dv, ds_out, dslopes, workspace, scale, drop, (hipStream_t)stream)))
}

}  // extern "C"
