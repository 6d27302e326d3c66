// libbptscore: launchers and C ABI (include/bptscore.h) of the fused attention with capped scores and distance: the MOD forms of the
// tile kernels in bpttiles.h.
#include "bpttiles.h"

#include "../../include/bptscore.h"

namespace {

// dslopes[head] = -(sum of the tiles' parts), a workgroup a head, in a fixed order; how many tiles there are stands in the plan
__global__ __launch_bounds__(BLOCK) void k_slope_finish(const float *__restrict__ part, const int32_t *__restrict__ n_groups, int heads, int parts,
                                                        float *__restrict__ dslopes) {
    __shared__ double meet[BLOCK];
    const int head = blockIdx.x, n = __builtin_amdgcn_readfirstlane(*n_groups) * parts;
    auto at = [&](int i) { return part[((size_t)(i / parts) * heads + head) * parts + i % parts]; };
    double x = 0.0;
    int i = threadIdx.x;
    for (; i + 7 * BLOCK < n; i += 8 * BLOCK) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = at(i + u * BLOCK);
#pragma unroll
        for (int u = 0; u < 8; ++u) x += v[u];
    }
    for (; i < n; i += BLOCK) x += at(i);
    meet[threadIdx.x] = x;
    for (int o = BLOCK / 2; o > 0; o >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < o) meet[threadIdx.x] += meet[threadIdx.x + o];
    }
    if (threadIdx.x == 0) dslopes[head] = (float)-meet[0];
}

// The scratch of the two backward kernels: (p, ds) of the edges, or in bfloat16 without a bias (lse, delta) of the rows
inline int64_t scratch_bytes(const bpt_plan *Pin, const bpt_plan *Pout, int h, int dtype, bool biased) {
    if (dtype == BPT_BF16 && !biased) return round16(std::max(Pin->n_rows, Pout->n_index_nodes) * h * 8);
    return round16(Pin->n_edges * h * (dtype == BPT_BF16 ? 4 : 8));
}
constexpr int MOST_PARTS = 4;
inline int64_t slope_bytes(const bpt_plan *Pin, int h) { return round16(Pin->n_groups * h * MOST_PARTS * 4); }

inline ScoreMod make_mod(const bpt_score *sc, float scale, bool entries_are_keys, float *part) {
    ScoreMod m{};
    if (sc->cap > 0.f) {
        m.to_tanh = scale / sc->cap;
        m.from_tanh = sc->cap * LOG2E;
    }
    m.slopes = sc->slopes;
    m.pos_member = entries_are_keys ? sc->pos_q : sc->pos_k;
    m.pos_entry = entries_are_keys ? sc->pos_k : sc->pos_q;
    m.part = part;
    return m;
}

// f(DROP, BIAS, SP) with compile-time values
template <typename F> void pick(bool drop, bool biased, int parts, F &&f) {
    using std::integral_constant;
    auto with_parts = [&](auto d, auto b) {
        if (parts == 4) f(d, b, integral_constant<int, 4>{});
        else if (parts == 2) f(d, b, integral_constant<int, 2>{});
        else f(d, b, integral_constant<int, 1>{});
    };
    auto with_bias = [&](auto d) {
        if (biased) with_parts(d, integral_constant<int, 1>{});
        else with_parts(d, integral_constant<int, 0>{});
    };
    if (drop) with_bias(integral_constant<bool, true>{});
    else with_bias(integral_constant<bool, false>{});
}

template <typename T, int H>
int run_forward(const bpt_plan *P, const bpt_score *sc, const void *q, const void *k, const void *v, const float *bias, void *o, float *lse, void *ws,
                float scale, Dropout drop, hipStream_t s) {
    constexpr int D = 64, HW = 4;
    float *ws_acc = (float *)ws, *ws_ml = ws_acc ? ws_acc + (size_t)P->n_slots * H * D : nullptr;
    const ScoreMod md = make_mod(sc, scale, true, nullptr);
    pick(drop.thr != 0, bias != nullptr, tile_parts(P, H, sizeof(T)), [&](auto dr, auto bi, auto sp) {
        const dim3 grid((unsigned)(group_grid(P) * (H * sp() / HW))), block(HW * WAVE);
        if constexpr (sizeof(T) == 4)
            hipLaunchKernelGGL((k_attn_fwd_tile<T, H, D, HW, dr(), bi(), false, sp(), true>), grid, block, 0, s, *P, (const T *)q, (const T *)k, (const T *)v,
                               (T *)o, lse, ws_acc, ws_ml, scale * LOG2E, drop.thr, drop.seed, drop.inv, bias, Narrow{}, Keep{}, md);
        else
            hipLaunchKernelGGL((k_attn_fwd_rows_bf16<H, D, HW, TILE_BF16_WPE, dr(), bi(), sp(), true>), grid, block, 0, s, *P, (const T *)q, (const T *)k,
                               (const T *)v, (T *)o, lse, ws_acc, ws_ml, scale * LOG2E, drop.thr, drop.seed, drop.inv, bias, md);
    });
    const int st = launch_status();
    if (st != BPT_OK || P->n_heavy == 0) return st;
    hipLaunchKernelGGL((k_attn_fwd_combine<T, H, D>), dim3((unsigned)P->n_heavy, H * D / WAVE), dim3(BLOCK), 0, s, P->heavy, (const float *)ws_acc,
                       (const float *)ws_ml, (T *)o, lse, Narrow{}, (T *)nullptr);
    return launch_status();
}

template <typename T, int H>
int run_backward(const bpt_plan *Pin, const bpt_plan *Pout, const bpt_score *sc, const void *q, const void *k, const void *v, const float *bias, const void *o,
                 const void *d_o, const float *lse, void *dq, void *dk, void *dv, float *ds_out, float *dslopes, void *ws, float scale, Dropout drop,
                 hipStream_t s) {
    constexpr int D = 64, HW = 4;
    const int dtype = sizeof(T) == 4 ? BPT_F32 : BPT_BF16;
    const bool biased = bias != nullptr, again = sizeof(T) == 2 && !biased;      // (bfloat16 forms (p, ds) again as the layer without options does)
    char *at = (char *)ws;
    void *scratch = at;
    at += scratch_bytes(Pin, Pout, H, dtype, biased);
    float *part = dslopes ? (float *)at : nullptr;
    at += slope_bytes(Pin, H);
    float *ws_dq = (float *)at, *ws_dk = ws_dq + (size_t)Pin->n_slots * H * D, *ws_dv = ws_dk + (size_t)Pout->n_slots * H * D;
    const int parts_in = tile_parts(Pin, H, sizeof(T)), parts_out = tile_parts(Pout, H, sizeof(T));
    const ScoreMod md = make_mod(sc, scale, true, part);
    pick(drop.thr != 0, biased, parts_in, [&](auto dr, auto bi, auto sp) {
        const dim3 grid((unsigned)(group_grid(Pin) * (H * sp() / HW))), block(HW * WAVE);
        if constexpr (sizeof(T) == 4)
            hipLaunchKernelGGL((k_attn_bwd_dst_tile<T, H, D, HW, dr(), bi(), false, sp(), true>), grid, block, 0, s, *Pin, (const T *)q, (const T *)k, (const T *)v,
                               (const T *)o, (const T *)d_o, lse, (T *)dq, (float2 *)scratch, ws_dq, scale, scale * LOG2E, drop.thr, drop.seed, drop.inv, bias,
                               ds_out, Narrow{}, md);
        else
            hipLaunchKernelGGL((k_attn_bwd_dst_rows_bf16<H, D, HW, TILE_BF16_WPE_DST, dr(), bi(), bi() != 0, sp(), true>), grid, block, 0, s, *Pin, (const T *)q,
                               (const T *)k, (const T *)v, (const T *)o, (const T *)d_o, lse, (T *)dq, (uint32_t *)scratch, (float2 *)scratch, ws_dq, scale,
                               scale * LOG2E, drop.thr, drop.seed, drop.inv, bias, ds_out, md);
    });
    int st = launch_status();
    if (st != BPT_OK) return st;
    pick(drop.thr != 0, biased, parts_out, [&](auto dr, auto bi, auto sp) {
        const dim3 grid((unsigned)(group_grid(Pout) * (H * sp() / HW))), block(HW * WAVE);
        if constexpr (sizeof(T) == 4)
            hipLaunchKernelGGL((k_attn_bwd_src_tile<T, H, D, HW, false, sp()>), grid, block, 0, s, *Pout, (const T *)q, (const T *)d_o, (const float2 *)scratch,
                               (T *)dk, (T *)dv, ws_dk, ws_dv, Narrow{});
        else if constexpr (bi() != 0)
            hipLaunchKernelGGL((k_attn_bwd_src_tile_bf16<H, D, HW, TILE_BF16_WPE_SRC, false, sp()>), grid, block, 0, s, *Pout, (const T *)q, (const T *)d_o,
                               (const uint32_t *)scratch, (T *)dk, (T *)dv, ws_dk, ws_dv, Narrow{});
        else
            hipLaunchKernelGGL((k_attn_bwd_src_tile_bf16_again<H, D, HW, TILE_BF16_WPE_AGAIN, dr(), sp(), true>), grid, block, 0, s, *Pout, (const T *)q,
                               (const T *)k, (const T *)v, (const T *)d_o, (const float2 *)scratch, (T *)dk, (T *)dv, ws_dk, ws_dv, scale, scale * LOG2E,
                               drop.thr, drop.seed, drop.inv, make_mod(sc, scale, false, nullptr));
    });
    st = launch_status();
    if (st != BPT_OK) return st;
    if (Pin->n_heavy + Pout->n_heavy > 0)
        hipLaunchKernelGGL((k_combine_sum3<T>), dim3((unsigned)(Pin->n_heavy + Pout->n_heavy), H * D / (4 * WAVE), 2), dim3(BLOCK), 0, s, Pin->heavy,
                           (int)Pin->n_heavy, (const float *)ws_dq, (T *)dq, Pout->heavy, (const float *)ws_dk, (T *)dk, (T *)dv, H * D,
                           (size_t)Pout->n_slots * H * D, Narrow{});
    if (dslopes) hipLaunchKernelGGL(k_slope_finish, dim3(H), dim3(BLOCK), 0, s, (const float *)part, Pin->grp_chunks + 8, H, parts_in, dslopes);
    return launch_status();
}

inline int check_score(const bpt_plan *P, const bpt_score *sc, int h, int dtype, float dropout_p, const float *bias) {
    const int st = check_plan(P, true);
    if (st != BPT_OK) return st;
    if (!sc) return BPT_ERR_NULL;
    if (dtype != BPT_F32 && dtype != BPT_BF16) return dtype == BPT_F64 ? BPT_ERR_UNSUPPORTED : BPT_ERR_DTYPE;
    if (h != 8 && h != 16 && !(h == 4 && dtype == BPT_F32)) return BPT_ERR_UNSUPPORTED;
    if (!(sc->cap >= 0.f && sc->cap <= 3.0e38f) || !(dropout_p >= 0.f && dropout_p < 1.f)) return BPT_ERR_SIZE;
    if (sc->slopes && (!sc->pos_q || !sc->pos_k)) return BPT_ERR_NULL;
    if (P->n_rows == 0 || P->n_groups == 0) return P->n_edges == 0 ? BPT_OK : BPT_ERR_UNSUPPORTED;
    if (!has_tiles(P, h, 64, dtype == BPT_BF16 ? 2 : 4)) return BPT_ERR_UNSUPPORTED;
    if ((bias || dropout_p > 0.f) && !P->grp_eids) return BPT_ERR_PLAN;
    if (bias && P->bias_by_pair) return BPT_ERR_PLAN;
    return BPT_OK;
}
inline bool on16(std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (!aligned16(p)) return false;
    return true;
}

#define DISPATCH(CALL)                                                   \
    if (dtype == BPT_F32) {                                              \
        using T = float;                                                 \
        if (h == 4) { constexpr int H = 4; return CALL; }                \
        if (h == 8) { constexpr int H = 8; return CALL; }                \
        { constexpr int H = 16; return CALL; }                           \
    } else {                                                             \
        using T = bf16_t;                                                \
        if (h == 8) { constexpr int H = 8; return CALL; }                \
        { constexpr int H = 16; return CALL; }                           \
    }

}  // namespace

extern "C" {

int64_t bpt_score_forward_workspace_bytes(const bpt_plan *plan_in, int h) {
    return plan_in && h > 0 ? round16(plan_in->n_slots * ((int64_t)h * 64 + 2 * h) * 4) : -1;
}

int64_t bpt_score_backward_workspace_bytes(const bpt_plan *plan_in, const bpt_plan *plan_out, int h, int dtype, int has_bias) {
    if (!plan_in || !plan_out || h < 1 || (dtype != BPT_F32 && dtype != BPT_BF16)) return -1;
    return scratch_bytes(plan_in, plan_out, h, dtype, has_bias != 0) + slope_bytes(plan_in, h) +
           round16((plan_in->n_slots + 2 * plan_out->n_slots) * (int64_t)h * 64 * 4);
}

int bpt_score_forward(const bpt_plan *plan_in, const bpt_score *score, const void *q, const void *k, const void *v, const float *bias, void *o, float *lse,
                      void *workspace, int64_t workspace_bytes, float scale, float dropout_p, uint64_t dropout_seed, int h, int dtype, void *stream) {
    const int st = check_score(plan_in, score, h, dtype, dropout_p, bias);
    if (st != BPT_OK) return st;
    if (plan_in->n_rows == 0) return BPT_OK;
    if (plan_in->n_groups == 0) return BPT_ERR_UNSUPPORTED;
    if (!q || !k || !v || !o || !lse) return BPT_ERR_NULL;
    if (!on16({q, k, v, o, workspace})) return BPT_ERR_UNSUPPORTED;
    const int64_t need = bpt_score_forward_workspace_bytes(plan_in, h);
    if (need > 0 && (!workspace || workspace_bytes < need)) return BPT_ERR_WORKSPACE;
    const Dropout drop = make_dropout(dropout_p, dropout_seed);
    DISPATCH((run_forward<T, H>(plan_in, score, q, k, v, bias, o, lse, workspace, scale, drop, (hipStream_t)stream)))
}

int bpt_score_backward(const bpt_plan *plan_in, const bpt_plan *plan_out, const bpt_score *score, const void *q, const void *k, const void *v,
                       const float *bias, const void *o, const void *d_o, const float *lse, void *dq, void *dk, void *dv, float *ds_out, float *dslopes,
                       void *workspace, int64_t workspace_bytes, float scale, float dropout_p, uint64_t dropout_seed, int h, int dtype, void *stream) {
    int st = check_score(plan_in, score, h, dtype, dropout_p, bias);
    if (st != BPT_OK) return st;
    st = check_plan(plan_out, true);
    if (st != BPT_OK) return st;
    if (plan_in->n_edges != plan_out->n_edges) return BPT_ERR_PLAN;
    if (plan_in->n_groups == 0 || !has_tiles(plan_out, h, 64, dtype == BPT_BF16 ? 2 : 4) || !plan_out->grp_pairs) return BPT_ERR_UNSUPPORTED;
    if ((bias != nullptr) != (ds_out != nullptr) || (dslopes && !score->slopes)) return BPT_ERR_NULL;
    if (dropout_p > 0.f && dtype == BPT_BF16 && !bias && !plan_out->grp_eids) return BPT_ERR_PLAN;
    if (!q || !k || !v || !o || !d_o || !lse || !dq || !dk || !dv) return BPT_ERR_NULL;
    if (!on16({q, k, v, o, d_o, dq, dk, dv, workspace})) return BPT_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < bpt_score_backward_workspace_bytes(plan_in, plan_out, h, dtype, bias != nullptr)) return BPT_ERR_WORKSPACE;
    const Dropout drop = make_dropout(dropout_p, dropout_seed);
    DISPATCH((run_backward<T, H>(plan_in, plan_out, score, q, k, v, bias, o, d_o, lse, dq, dk, dv, ds_out, dslopes, workspace, scale, drop, (hipStream_t)stream)))
}

}  // extern "C"
