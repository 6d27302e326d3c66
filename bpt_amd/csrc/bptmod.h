// What libbptscore and libbptbias share: the launchers of the fused attention with score options (capped scores, distance), with and without a bias by buckets: the MOD
// forms of the tile kernels in bpttiles.h.
#pragma once
#include "bpttiles.h"

#include "../../include/bptscore.h"

namespace {

// Split rows, a workgroup each, from the sums of their segments (bfloat16, comment at k_attn_bwd_dst_rows_bf16): delta of the row to the source side,
// and, fix[split row][head], (delta' - delta) and what the slopes' gradient gains by it.  float32 and with a score term (no stat): the latter alone, of the sum of ds that should be zero.
__global__ __launch_bounds__(BLOCK) void k_score_split(const int32_t *__restrict__ heavy, const float4 *__restrict__ split, float2 *__restrict__ stat,
                                                       float2 *__restrict__ fix, int heads) {
    __shared__ float4 meet[BLOCK];
    const int row = heavy[3 * blockIdx.x], s0 = heavy[3 * blockIdx.x + 1], ns = heavy[3 * blockIdx.x + 2];
    const int head = threadIdx.x % heads, lane = threadIdx.x / heads, lanes = BLOCK / heads;      // (8 or 16 heads)
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = lane; i < ns; i += lanes) {
        const float4 y = split[(size_t)(s0 + i) * heads + head];
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
    }
    meet[threadIdx.x] = x;
    for (int o = lanes / 2; o > 0; o >>= 1) {
        __syncthreads();
        if (lane < o) {
            const float4 y = meet[threadIdx.x + o * heads];
            x.x += y.x;
            x.y += y.y;
            x.z += y.z;
            meet[threadIdx.x] = x;
        }
    }
    if (lane == 0 && !stat) fix[(size_t)blockIdx.x * heads + head] = make_float2(0.f, x.z == 0.f ? 0.f : -x.x / x.z * x.y);
    if (lane == 0 && stat) {
        float2 *const at = stat + (size_t)row * heads + head;
        const float delta = at->y, better = x.z == 0.f ? delta : x.x / x.z, less = delta == delta ? delta - better : 0.f;
        fix[(size_t)blockIdx.x * heads + head] = make_float2(less, less * x.y);
        at->y = better;
    }
}

// dslopes[head] = -(sum of the tiles' parts and of what split rows gained), by a workgroup, in a fixed order; how many tiles there are stands in the plan
struct SlopeSum {
    const float *part;                 // [group][head][part]
    const int32_t *n_groups;
    int heads, parts;                  // as part counts them
    const float2 *fix;                 // [split row][head], the second of the two
    int n_fix, wanted;                 // heads to sum up, or 0
    float *dslopes;
};
__device__ __forceinline__ void slope_sum_block(const SlopeSum &m, int head) {
    __shared__ double meet[BLOCK];
    const int n = __builtin_amdgcn_readfirstlane(*m.n_groups) * m.parts;
    auto at = [&](int i) { return m.part[((size_t)(i / m.parts) * m.heads + head) * m.parts + i % m.parts]; };
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
    for (i = threadIdx.x; i < m.n_fix; i += BLOCK) x += m.fix[(size_t)i * m.heads + head].y;
    meet[threadIdx.x] = x;
    for (int o = BLOCK / 2; o > 0; o >>= 1) {
        __syncthreads();
        if ((int)threadIdx.x < o) meet[threadIdx.x] += meet[threadIdx.x + o];
    }
    if (threadIdx.x == 0) m.dslopes[head] = (float)-meet[0];
}

// dq of a split row, 128 columns (blockIdx.y, blockIdx.z): the sum of its segments' and (delta' - delta) times that of what they left of p du K; half wavefront i
// takes segments i, i + 8, ..., up to eight in flight
template <bool NARROW>
__device__ __forceinline__ void merge_dq_block(const int32_t *__restrict__ hv, const float *__restrict__ ws, const bf16_t *__restrict__ low,
                                               const float2 *__restrict__ fix, bf16_t *__restrict__ dq, int C, const Narrow &nw) {
    constexpr int HALVES = 2 * WAVES_PER_BLOCK;
    __shared__ float4 part[2][HALVES][WAVE / 2];
    const int row = hv[0], s0 = hv[1], ns = hv[2];
    const int lane = threadIdx.x & 31, half = threadIdx.x >> 5, j = (((int)blockIdx.y * 2 + (int)blockIdx.z) * 32 + lane) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f), b = s;
    const size_t first = (size_t)s0 * C + j;
    int k = half;
    auto take = [&](auto n) {
        float4 t[n()];
        uint2 u[n()];
#pragma unroll
        for (int i = 0; i < n(); ++i) {
            const size_t at = first + (size_t)(k + i * HALVES) * C;
            t[i] = *reinterpret_cast<const float4 *>(ws + at);
            u[i] = *reinterpret_cast<const uint2 *>(low + at);
        }
        issue_loads_first();
#pragma unroll
        for (int i = 0; i < n(); ++i) {
            const float4 y = tile_four(u[i]);
            s.x += t[i].x; s.y += t[i].y; s.z += t[i].z; s.w += t[i].w;
            b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
        }
        k += n() * HALVES;
    };
    while (k + 7 * HALVES < ns) take(std::integral_constant<int, 8>{});
    if (k + 3 * HALVES < ns) take(std::integral_constant<int, 4>{});
    if (k + HALVES < ns) take(std::integral_constant<int, 2>{});
    if (k < ns) take(std::integral_constant<int, 1>{});
    part[0][half][lane] = s;
    part[1][half][lane] = b;
    __syncthreads();
    if (half != 0) return;
    s = part[0][0][lane];
    b = part[1][0][lane];
#pragma unroll
    for (int i = 1; i < HALVES; ++i) {
        const float4 x = part[0][i][lane], y = part[1][i][lane];
        s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
        b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
    }
    const int head = j >> 6, col = j & 63;
    const float less = fix[head].x;
    const float x[4] = {fmaf(less, b.x, s.x), fmaf(less, b.y, s.y), fmaf(less, b.z, s.z), fmaf(less, b.w, s.w)};
    if constexpr (NARROW) {                                       // 64 columns of the partials per head, d of the result
        bf16_t *const at = dq + (size_t)row * (nw.heads * nw.d) + head * nw.d + col;
        for (int e = 0; e < 4; ++e)
            if (head < nw.heads && col + e < nw.d) Elem<bf16_t>::st(at + e, x[e]);
    } else {
        store4<bf16_t>(dq + (size_t)row * C + j, make_float4(x[0], x[1], x[2], x[3]));
    }
}

// The backward's last launch: k_combine_sum3's sums of split rows (dq; dk and dv) and, in workgroups of their own in front of them, the slopes' gradient, which
// as a launch by itself cost 4 us (8 at L = 32768, k = 8).  Grid (m.wanted + n_a + n_b, C / 256, 2).
template <typename T, bool NARROW>
__global__ __launch_bounds__(BLOCK) void k_score_merge(SlopeSum m, const int32_t *__restrict__ heavy_a, int n_a, const float *__restrict__ ws_a,
                                                       const bf16_t *__restrict__ low, T *__restrict__ YA, const int32_t *__restrict__ heavy_b,
                                                       const float *__restrict__ ws_b, T *__restrict__ YB0, T *__restrict__ YB1, int C, size_t ws_stride_b, Narrow nw) {
    const int x = (int)blockIdx.x - m.wanted;
    if (x < 0) {
        if (blockIdx.y == 0 && blockIdx.z == 0) slope_sum_block(m, (int)blockIdx.x);
    } else if (x < n_a) {
        if constexpr (sizeof(T) == 2) {
            if (low) return merge_dq_block<NARROW>(heavy_a + 3 * x, ws_a, low, m.fix + (size_t)x * m.heads, YA, C, nw);
        }
        if (blockIdx.z == 0) combine_sum_block4<T, NARROW>(heavy_a + 3 * x, ws_a, YA, C, false, -1, nw);
    } else {
        combine_sum_block4<T, NARROW>(heavy_b + 3 * (x - n_a), ws_b + (size_t)blockIdx.z * ws_stride_b, blockIdx.z == 0 ? YB0 : YB1, C, false, -1, nw);
    }
}
template <typename T, bool NARROW>
int run_merge(const SlopeSum &m, const bpt_plan *Pin, const bpt_plan *Pout, const float *ws_dq, const bf16_t *low, T *dq, const float *ws_dk, T *dk, T *dv, int C, const Narrow &nw,
              hipStream_t s) {
    const unsigned blocks = (unsigned)(m.wanted + Pin->n_heavy + Pout->n_heavy);
    if (blocks == 0) return BPT_OK;
    hipLaunchKernelGGL((k_score_merge<T, NARROW>), dim3(blocks, Pin->n_heavy + Pout->n_heavy > 0 ? C / (4 * WAVE) : 1, Pin->n_heavy + Pout->n_heavy > 0 ? 2 : 1), dim3(BLOCK), 0,
                       s, m, Pin->heavy, (int)Pin->n_heavy, ws_dq, low, dq, Pout->heavy, ws_dk, dk, dv, C, (size_t)Pout->n_slots * C, nw);
    return launch_status();
}

// Forward of few query rows (a decoder that takes one token at a time): a tile would walk a row's neighbours in one chain with fifteen of its sixteen
// rows empty.  Here a workgroup of NW wavefronts has a row or a segment of one, a wavefront whole rows of K and V, lane l columns of head l / (64 / H), four
// edges in flight, and the segments are merged as those of the tiles' split rows.  Without dropout and score term.
template <typename T, int H, int D, int BATCH, int NW, bool BUCKETS = false>
__global__ __launch_bounds__(NW == 1 ? BLOCK : NW * WAVE) void k_score_fwd_rows(bpt_plan P, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                                                                                T *__restrict__ o, float *__restrict__ lse, float *__restrict__ ws_acc,
                                                                                float *__restrict__ ws_ml, float scale_log2e, typename ModArg<true, BUCKETS>::type md) {
    using L = Lay<T, H, D>;
    Item it;
    int part, parts;
    if (!fetch_item_part<NW, BATCH>(P, it, part, parts)) return;
    const int lane = threadIdx.x & 63, head = lane / L::LPH;
    float qv[L::EPL], acc[L::EPL];
    load_row<T, H, D>(q + (size_t)it.row * L::C, lane, qv);
#pragma unroll
    for (int i = 0; i < L::EPL; ++i) acc[i] = 0.f;
    const float slope = md.slopes ? md.slopes[head] * LOG2E : 0.f, pos_m = md.slopes ? md.pos_member[it.row] : 0.f;
    float m = m_init<true>(), l = 0.f;
    for (int p0 = it.begin; p0 < it.end; p0 += WAVE) {
        const int cnt = min(WAVE, it.end - p0);
        const int my_idx = lane < cnt ? P.idx[p0 + lane] : 0;
        const float my_pos = md.slopes && lane < cnt ? md.pos_entry[my_idx] : 0.f;
        int my_code = 0;
        if constexpr (BUCKETS) my_code = lane < cnt ? md.codes[p0 + lane] : 0;
        for (int b = 0; b < cnt; b += BATCH) {
            float kv[BATCH][L::EPL], vv[BATCH][L::EPL], x[BATCH], pos_e[BATCH], s[BATCH], du[BATCH], bz[BUCKETS ? BATCH : 1];
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int j = (b + e < cnt) ? b + e : b, src = __builtin_amdgcn_readlane(my_idx, j);
                pos_e[e] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(my_pos), j));
                load_row<T, H, D>(k + (size_t)src * L::C, lane, kv[e]);
                load_row<T, H, D>(v + (size_t)src * L::C, lane, vv[e]);
                if constexpr (BUCKETS) bz[e] = md.table[head * 256 + __builtin_amdgcn_readlane(my_code, j)];
            }
            issue_loads_first();
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                x[e] = head_sum<L::LPH>(dot_n<L::EPL>(qv, kv[e]));
                if constexpr (BUCKETS) x[e] += bz[e];
            }
            tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, s, du);
            float mx = m;
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                s[e] = (b + e < cnt) ? s[e] : -INFINITY;
                mx = fmaxf(mx, s[e]);
            }
            const float alpha = __builtin_amdgcn_exp2f(m - mx);
            l *= alpha;
#pragma unroll
            for (int i = 0; i < L::EPL; ++i) acc[i] *= alpha;
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const float pe = __builtin_amdgcn_exp2f(s[e] - mx);
                l += pe;
#pragma unroll
                for (int i = 0; i < L::EPL; ++i) acc[i] = fmaf(pe, vv[e][i], acc[i]);
            }
            m = mx;
        }
    }
    if constexpr (NW > 1) {
        __shared__ float held[NW - 1][L::EPL + 2][WAVE];
        if (part > 0 && part < parts) {
#pragma unroll
            for (int i = 0; i < L::EPL; ++i) held[part - 1][i][lane] = acc[i];
            held[part - 1][L::EPL][lane] = m;
            held[part - 1][L::EPL + 1][lane] = l;
        }
        __syncthreads();
        if (part > 0) return;
        for (int w = 0; w < parts - 1; ++w) {
            const float mw = held[w][L::EPL][lane], mx = fmaxf(m, mw);
            const float a = __builtin_amdgcn_exp2f(m - mx), b = __builtin_amdgcn_exp2f(mw - mx);
            l = fmaf(b, held[w][L::EPL + 1][lane], a * l);
#pragma unroll
            for (int i = 0; i < L::EPL; ++i) acc[i] = fmaf(b, held[w][i][lane], a * acc[i]);
            m = mx;
        }
    }
    if (it.slot < 0) {
        const float inv = has_sum<true>(l) ? 1.f / l : 0.f;
#pragma unroll
        for (int i = 0; i < L::EPL; ++i) acc[i] *= inv;
        store_row<T, H, D>(o + (size_t)it.row * L::C, lane, acc);
        if (lane % L::LPH == 0) lse[(size_t)it.row * H + head] = has_sum<true>(l) ? m + log2f(l) : 0.f;
    } else {
        store_row_ws<T, H, D>(ws_acc + (size_t)it.slot * L::C, lane, acc);
        if (lane % L::LPH == 0) {
            ws_ml[((size_t)it.slot * H + head) * 2] = m;
            ws_ml[((size_t)it.slot * H + head) * 2 + 1] = l;
        }
    }
}

// bfloat16 heads of fewer than 64 columns, read as they are (Narrow in bpttiles.h): the two sides of the backward, k_attn_bwd_dst_rows_bf16 and
// k_attn_bwd_src_tile_bf16_again with rows of 8 bytes a lane, kept in registers for the products over the entries and turned in LDS for those over the
// columns.  delta comes from the pairs in 32 bits, as there, so p and ds are formed twice rather than handed over in 16 bits each.
// Bound by the loads' latency (a block's rows are asked for when it begins, three or four wavefronts a SIMD cover for one another; compiled for three or four,
// either side is level, four spills the source side).  8192 tokens, k = 4, 6 x 50 bfloat16: 22.6 + 25.7 us, the training pass 102.7 us of which 81 are kernels;
// on copies padded to 8 x 64 the pass took 208.  12 x 64: 49 + 50 us, the pass 157, on copies 298.
constexpr int NARROW_WPE_DST = 3, NARROW_WPE_SRC = 3;
template <int HW, bool DROP, int SP>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(NARROW_WPE_DST))) void k_score_bwd_dst_narrow_bf16(
    bpt_plan P, const bf16_t *__restrict__ q, const bf16_t *__restrict__ k, const bf16_t *__restrict__ v, const bf16_t *__restrict__ o,
    const bf16_t *__restrict__ d_o, const float *__restrict__ lse, bf16_t *__restrict__ dq, float2 *__restrict__ stat, float *__restrict__ ws_dq, float scale,
    float scale_log2e, uint32_t drop_thr, uint32_t drop_seed, float drop_inv, Narrow nw, ScoreMod md) {
    constexpr int H = 16, D = 64;
    const int Hs = nw.h;
    const uint32_t RB = (uint32_t)(nw.heads * nw.d) * 2;
    TileCtx t;
    if (!tile_begin<bf16_t, H, D, HW, true, SP>(P, t, nw)) return;
    __shared__ int2 ent_lds[HW][TILE_CHUNK];
    int2 *const ent = ent_lds[t.wv];
    constexpr int PIECE = SP > 1 ? TILE_PART_FLOATS : TILE_KT_FLOATS_BF16;
    static_assert(PIECE >= TILE_KT_FLOATS_BF16, "the rows fit");
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    __shared__ __attribute__((aligned(16))) float pos_lds[HW][TILE_R];
    char *const kt = reinterpret_cast<char *>(piece[t.wv]);
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const uint32_t offc = t.offv;
    const char *kb = reinterpret_cast<const char *>(k), *vb = reinterpret_cast<const char *>(v);
    const size_t mrow = (size_t)max(t.member.x, 0) * RB + t.offa, at = (size_t)max(t.member.x, 0) * Hs + t.head;
    Bf8 qb[2], dob[2];
    float delta = 0.f;
    {
        Bf8 ob[2];
        tile_load_row_bf16(reinterpret_cast<const char *>(q) + mrow, qb, g, nw);
        tile_load_row_bf16(reinterpret_cast<const char *>(d_o) + mrow, dob, g, nw);
        tile_load_row_bf16(reinterpret_cast<const char *>(o) + mrow, ob, g, nw);
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
            const uint32_t a[4] = {dob[h2].q.x, dob[h2].q.y, dob[h2].q.z, dob[h2].q.w}, b[4] = {ob[h2].q.x, ob[h2].q.y, ob[h2].q.z, ob[h2].q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                delta = fmaf(__uint_as_float(a[i] << 16), __uint_as_float(b[i] << 16), delta);
                delta = fmaf(__uint_as_float(a[i] & 0xffff0000u), __uint_as_float(b[i] & 0xffff0000u), delta);
            }
        }
        delta = groups_sum(delta);                                // dO . O of member c, this head
    }
    const float lse_c = lse[at];
    float slope = 0.f, pos_m = 0.f, slope_sum = 0.f, dp_sum = 0.f, far_sum = 0.f, p_sum = 0.f;
    if (md.slopes) {
        slope = md.slopes[t.head] * LOG2E;
        pos_m = md.pos_member[max(t.member.x, 0)];
    }
    floatx4v acc[4], pk[4];                                       // pk: sum of p du K
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) { acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; pk[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
    struct Blk {
        uint2 kc[4], vc[4];                                       // columns 4 c .. 4 c + 3 of the K / V rows of entries 4 g + r
        int mk[4];                                                // bit c of mk[r]: the pair (entry 4 g + r, member c) exists
        int xe[DROP ? 4 : 1];
        float pos;                                                // of entry c, in the first lane group
    };
    auto walk = [&](auto again) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(again)::value;
    if constexpr (CAREFUL) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        if (p0 != t.p_begin) tile_ask_entries(P, p0, cnt, t.lane, er);
        tile_put_entries(er, ent, cnt, t.lane);
        auto issue = [&](Blk &B, int b) {
            if constexpr (DROP) tile_pair_eids(P, p0 + TILE_R * b + 4 * g, t.p_end, c, B.xe);
            if (md.slopes && g == 0) B.pos = md.pos_entry[ent[TILE_R * b + c].x];
            const int4 e01 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g]);
            const int4 e23 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g + 2]);
            const int idxv[4] = {e01.x, e01.z, e23.x, e23.z};
            B.mk[0] = e01.y; B.mk[1] = e01.w; B.mk[2] = e23.y; B.mk[3] = e23.w;
#pragma unroll
            for (int r = 0; r < 4; ++r) B.kc[r] = tile_row4_bf16<true>(kb + ((uint32_t)idxv[r] * RB + offc));
#pragma unroll
            for (int r = 0; r < 4; ++r) B.vc[r] = tile_row4_bf16<true>(vb + ((uint32_t)idxv[r] * RB + offc));
        };
        auto compute = [&](const Blk &B) {
            if (md.slopes && g == 0) pos_lds[t.wv][c] = B.pos;
            Bf8 row[2];
            tile_rows_to_operand_bf16(kt, B.kc, c, g, row, nw);
            const floatx4v st = tile_dot_bf16(row, qb);
            tile_rows_to_operand_bf16(kt, B.vc, c, g, row, nw);
            const floatx4v dp = tile_dot_bf16(row, dob);
            const floatx4v at_e = *reinterpret_cast<const floatx4v *>(&pos_lds[t.wv][4 * g]);
            const float pos_e[4] = {at_e[0], at_e[1], at_e[2], at_e[3]}, x[4] = {st[0], st[1], st[2], st[3]};
            float sm[4], du[4], ds[4], pdu[4];
            tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, sm, du);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float pe = where_pair_or_zero(B.mk[r], c, __builtin_amdgcn_exp2f(sm[r] - lse_c));
                float mt = 1.f;                                   // dropout multiplier of this pair (as in the forward)
                if constexpr (DROP) mt = dropout_keep((uint32_t)B.xe[DROP ? r : 0] * (uint32_t)Hs + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
                const float y = where_pair_or_zero(B.mk[r], c, pe * (dp[r] * mt));
                ds[r] = fmaf(-pe, delta, y);
                dp_sum += y;
                p_sum += pe;
                if (md.part) {
                    const float far = fabsf(pos_m - pos_e[r]);
                    slope_sum += pair_if<CAREFUL>(B.mk[r], c, ds[r] * far);
                    far_sum += pair_if<CAREFUL>(B.mk[r], c, pe * far);
                }
                ds[r] = pair_if<CAREFUL>(B.mk[r], c, ds[r] * du[r]);
                pdu[r] = pair_if<CAREFUL>(B.mk[r], c, pe * du[r]);
            }
            if constexpr (CAREFUL) {
                tile_axpy_pairs(ds, B.mk, B.kc, c, g, acc);
                tile_axpy_pairs(pdu, B.mk, B.kc, c, g, pk);
            } else {
                Bf4 da;
                da.u[0] = pack_bf16(ds[0], ds[1]);
                da.u[1] = pack_bf16(ds[2], ds[3]);
                tile_axpy_bf16(da, B.kc, acc);
                da.u[0] = pack_bf16(pdu[0], pdu[1]);
                da.u[1] = pack_bf16(pdu[2], pdu[3]);
                tile_axpy_bf16(da, B.kc, pk);
            }
        };
        tile_walk<Blk>(nblk, issue, compute);
        wave_lds_fence();
    }
    };
    walk(std::false_type{});
    if (tile_any_odd(tile_odd(acc) + tile_odd(pk) + (slope_sum + far_sum) * 0.f)) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) { acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; pk[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
            slope_sum = far_sum = dp_sum = p_sum = 0.f;
            walk(std::true_type{});
    }
    float4 sums = make_float4(groups_sum(dp_sum), groups_sum(far_sum), groups_sum(p_sum), 0.f);      // of member c, of this part
    if constexpr (SP > 1) {
        __shared__ float4 meet[HW][TILE_R];
        tile_parts_sum<SP, HW>(meet, t, sums);
    }
    const bool segment = t.member.y >= 0;
    const float better = segment || sums.z == 0.f ? delta : sums.x / sums.z, less = delta == delta ? delta - better : 0.f;      // (as in k_attn_bwd_dst_rows_bf16)
    slope_sum = fmaf(less, far_sum, slope_sum);
    // (lane (c, g) of the sums holds members 4 g + r, less is member c's)
    float less_m[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) less_m[r] = lane_bcast(less, 4 * g + r);
#pragma unroll
    for (int nb = 0; nb < 4; ++nb)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[nb][r] = fmaf(less_m[r], pk[nb][r], acc[nb][r]);
    if (g == 0 && t.part == 0 && t.member.x >= 0) {
        stat[at] = make_float2(lse_c, better);
        if (segment) md.split[(size_t)t.member.y * Hs + t.head] = sums;
    }
    if (__builtin_amdgcn_ballot_w64(segment) != 0) tile_put_low<SP, H, D, true>(md, t, piece[t.wv], piece[t.wv % (HW / SP)], (HW / SP) * PIECE, pk, nw);
    tile_put_slope_part<SP>(md, t, Hs, slope_sum);
    if constexpr (SP > 1) {
        tile_park(piece[t.wv], acc, t.lane);
        __syncthreads();
        tile_meet_and_store<SP, H, D, true>(piece[t.wv % (HW / SP)], (HW / SP) * PIECE, t, dq, ws_dq, nw);
    } else {
        tile_store_rows<H, D, false, true>(t, acc, 1.f, dq, ws_dq, nw);
    }
}

template <int HW, bool DROP, int SP>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(NARROW_WPE_SRC))) void k_score_bwd_src_narrow_bf16(
    bpt_plan P, const bf16_t *__restrict__ q, const bf16_t *__restrict__ k, const bf16_t *__restrict__ v, const bf16_t *__restrict__ d_o,
    const float2 *__restrict__ stat, bf16_t *__restrict__ dk, bf16_t *__restrict__ dv, float *__restrict__ ws_dk, float *__restrict__ ws_dv, float scale,
    float scale_log2e, uint32_t drop_thr, uint32_t drop_seed, float drop_inv, Narrow nw, ScoreMod md) {
    constexpr int H = 16, D = 64;
    const int Hs = nw.h;
    const uint32_t RB = (uint32_t)(nw.heads * nw.d) * 2;
    TileCtx t;
    if (!tile_begin<bf16_t, H, D, HW, true, SP>(P, t, nw)) return;
    // a wavefront's piece: its entry list, the rows being turned, the entries' (lse, delta) and positions; afterwards (SP > 1) what it has summed up
    constexpr int ENT = TILE_CHUNK * 2, STAT = ENT + TILE_KT_FLOATS_BF16, LIVE = STAT + 3 * TILE_R, PIECE = SP > 1 && 2 * TILE_PART_FLOATS > LIVE ? 2 * TILE_PART_FLOATS : LIVE;
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    int2 *const ent = reinterpret_cast<int2 *>(piece[t.wv]);
    char *const kt = reinterpret_cast<char *>(piece[t.wv] + ENT);
    float2 *const st_lds = reinterpret_cast<float2 *>(piece[t.wv] + STAT);
    float *const pos_lds = piece[t.wv] + STAT + 2 * TILE_R;
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const uint32_t offc = t.offv;
    const char *qb = reinterpret_cast<const char *>(q), *db = reinterpret_cast<const char *>(d_o);
    const float2 *const stat_h = stat + t.head;
    const size_t mrow = (size_t)max(t.member.x, 0) * RB + t.offa;
    Bf8 kr[2], vr[2];
    tile_load_row_bf16(reinterpret_cast<const char *>(k) + mrow, kr, g, nw);
    tile_load_row_bf16(reinterpret_cast<const char *>(v) + mrow, vr, g, nw);
    float slope = 0.f, pos_m = 0.f;
    if (md.slopes) {
        slope = md.slopes[t.head] * LOG2E;
        pos_m = md.pos_member[max(t.member.x, 0)];
    }
    floatx4v ak[4], av[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) { ak[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; av[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
    struct Blk {
        uint2 qr[4], dr[4];
        float2 ld;                                                // (lse, delta) of entry c, in the first lane group
        int mk[4];                                                // bit c of mk[r]: the pair (entry 4 g + r, member c) exists
        int xe[DROP ? 4 : 1];
        float pos;                                                // of entry c, in the first lane group
    };
    auto walk = [&](auto again) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(again)::value;
    if constexpr (CAREFUL) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        if (p0 != t.p_begin) tile_ask_entries(P, p0, cnt, t.lane, er);
        tile_put_entries(er, ent, cnt, t.lane);
        auto issue = [&](Blk &B, int b) {
            if constexpr (DROP) tile_pair_eids(P, p0 + TILE_R * b + 4 * g, t.p_end, c, B.xe);
            if (g == 0) {
                const int at = ent[TILE_R * b + c].x;
                B.ld = stat_h[(size_t)at * Hs];
                if (md.slopes) B.pos = md.pos_entry[at];
            }
            const int4 e01 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g]);
            const int4 e23 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g + 2]);
            const int idxv[4] = {e01.x, e01.z, e23.x, e23.z};
            B.mk[0] = e01.y; B.mk[1] = e01.w; B.mk[2] = e23.y; B.mk[3] = e23.w;
#pragma unroll
            for (int r = 0; r < 4; ++r) B.qr[r] = tile_row4_bf16<true>(qb + ((uint32_t)idxv[r] * RB + offc));
#pragma unroll
            for (int r = 0; r < 4; ++r) B.dr[r] = tile_row4_bf16<true>(db + ((uint32_t)idxv[r] * RB + offc));
        };
        auto compute = [&](const Blk &B) {
            if (g == 0) {
                st_lds[c] = B.ld;
                if (md.slopes) pos_lds[c] = B.pos;
            }
            Bf8 row[2];
            tile_rows_to_operand_bf16(kt, B.qr, c, g, row, nw);
            const floatx4v st = tile_dot_bf16(row, kr);
            tile_rows_to_operand_bf16(kt, B.dr, c, g, row, nw);
            const floatx4v dp = tile_dot_bf16(row, vr);
            const floatx4v l01 = *reinterpret_cast<const floatx4v *>(&st_lds[4 * g]), l23 = *reinterpret_cast<const floatx4v *>(&st_lds[4 * g + 2]);
            const float lse_e[4] = {l01[0], l01[2], l23[0], l23[2]}, delta_e[4] = {l01[1], l01[3], l23[1], l23[3]};
            const floatx4v at_e = *reinterpret_cast<const floatx4v *>(&pos_lds[4 * g]);
            const float pos_e[4] = {at_e[0], at_e[1], at_e[2], at_e[3]}, x[4] = {st[0], st[1], st[2], st[3]};
            float sm[4], du[4], pe[4], ds[4];
            tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, sm, du);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float p = where_pair_or_zero(B.mk[r], c, __builtin_amdgcn_exp2f(sm[r] - lse_e[r]));
                float mt = 1.f;                                   // dropout multiplier of this pair (as in the forward)
                if constexpr (DROP) mt = dropout_keep((uint32_t)B.xe[DROP ? r : 0] * (uint32_t)Hs + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
                ds[r] = where_pair_or_zero(B.mk[r], c, p * (dp[r] * mt - delta_e[r]) * du[r]);
                pe[r] = p * mt;
            }
            if constexpr (CAREFUL) {
                tile_axpy_pairs(ds, B.mk, B.qr, c, g, ak);
                tile_axpy_pairs(pe, B.mk, B.dr, c, g, av);
            } else {
                Bf4 pa, da;
                da.u[0] = pack_bf16(ds[0], ds[1]); da.u[1] = pack_bf16(ds[2], ds[3]);
                pa.u[0] = pack_bf16(pe[0], pe[1]); pa.u[1] = pack_bf16(pe[2], pe[3]);
                tile_axpy_bf16(da, B.qr, ak);
                tile_axpy_bf16(pa, B.dr, av);
            }
        };
        tile_walk<Blk>(nblk, issue, compute);
        wave_lds_fence();
    }
    };
    walk(std::false_type{});
    if (tile_any_odd(tile_odd(ak) + tile_odd(av))) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) { ak[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; av[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
            walk(std::true_type{});
    }
    if constexpr (SP > 1) {
        constexpr int NEXT = (HW / SP) * PIECE;
        tile_park(piece[t.wv], ak, t.lane);
        tile_park(piece[t.wv] + TILE_PART_FLOATS, av, t.lane);
        __syncthreads();
        const float *const part0 = piece[t.wv % (HW / SP)];
        tile_meet_and_store<SP, H, D, true>(part0, NEXT, t, dk, ws_dk, nw);
        tile_meet_and_store<SP, H, D, true>(part0 + TILE_PART_FLOATS, NEXT, t, dv, ws_dv, nw);
    } else {
        tile_store_rows<H, D, false, true>(t, ak, 1.f, dk, ws_dk, nw);
        tile_store_rows<H, D, false, true>(t, av, 1.f, dv, ws_dv, nw);
    }
}

// The scratch of the two backward kernels: (p, ds) of the edges, or in bfloat16 without a bias (lse, delta) of the rows
inline int64_t scratch_bytes(const bpt_plan *Pin, const bpt_plan *Pout, int h, int dtype, bool biased) {
    if (dtype == BPT_BF16 && !biased) return round16(std::max(Pin->n_rows, Pout->n_index_nodes) * h * 8);
    return round16(Pin->n_edges * h * (dtype == BPT_BF16 ? 4 : 8));
}
constexpr int MOST_PARTS = 4;
inline int64_t slope_bytes(const bpt_plan *Pin, int h) { return round16(Pin->n_groups * h * MOST_PARTS * 4); }
// bfloat16's segments: [slot][head] sums, [slot][column] of p du K, [split row][head] of k_score_split
struct SplitSums {
    float4 *sums;
    bf16_t *low;
    float2 *fix;
};
inline int64_t split_slot_bytes(int h, bool low) { return h * (16 + (low ? 64 * 2 : 0)); }
inline SplitSums split_sums(char *at, const bpt_plan *Pin, int h, bool low) {
    return SplitSums{(float4 *)at, low ? (bf16_t *)(at + Pin->n_slots * h * 16) : nullptr, (float2 *)(at + Pin->n_slots * split_slot_bytes(h, low))};
}
inline int64_t split_bytes(const bpt_plan *Pin, int h, bool low) { return Pin->n_slots * split_slot_bytes(h, low) + round16(Pin->n_heavy * h * 8); }
// Whether split rows' sums are looked at: bfloat16's always, for delta (again) or, with a score term, for the slopes' gradient, which a delta from o as stored puts off
// by more than itself where the long rows' parts cancel (L = 8192, 127 split rows, 1.1e-5 of the sum of its terms' absolute values, 1.1e-9 with them; the launch: a
// training pass 173.6 -> 176.5 us).
// float32's, a launch of 5 us for the slopes' gradient alone, where they are half of the rows or more (few queries of a long memory: 101 rows of 185 keys
// 1.1e-6 -> 6e-7 off).  Of a graph with few of them they carry little there: L = 8192, 127 split rows, 2.7e-7 without.
inline bool split_counts(const bpt_plan *Pin, bool again, bool slopes, bool rounded) {
    return Pin->n_heavy > 0 && (again || (slopes && (rounded || 2 * Pin->n_heavy >= Pin->n_rows)));
}

inline ScoreMod make_mod(const bpt_score *sc, float scale, bool entries_are_keys, float *part) {
    ScoreMod m{};
    m.scale = scale;
    if (sc->cap > 0.f) {
        const double to = (double)scale / sc->cap, w = to * to, base2 = (double)scale * 1.4426950408889634;
        m.to_tanh = (float)to;
        m.from_tanh = sc->cap * LOG2E;
        m.slope_of = (float)(-(double)scale / ((double)m.from_tanh * m.from_tanh));
        m.c[0] = (float)(-0.333331435918808 * w * base2);
        m.c[1] = (float)(0.13325878977775574 * w * w * base2);
        m.c[2] = (float)(-0.05304549261927605 * w * w * w * base2);
        m.c[3] = (float)(0.01724148355424404 * w * w * w * w * base2);
        m.far = (float)(0.25 / w);
    }
    m.slopes = sc->slopes;
    m.pos_member = entries_are_keys ? sc->pos_q : sc->pos_k;
    m.pos_entry = entries_are_keys ? sc->pos_k : sc->pos_q;
    m.part = part;
    return m;
}

// What a bias by buckets adds to a call's score options (BucketMod): the codes of either side's places, the heads' tables, and where bfloat16's source side leaves ds.
struct BucketArgs {
    const uint8_t *codes_in, *codes_out;
    const float *table;
    float *ds;
};
template <bool BUCKETS> inline typename ModArg<true, BUCKETS>::type with_buckets(const ScoreMod &m, const BucketArgs *b, bool entries_are_keys) {
    if constexpr (BUCKETS) {
        BucketMod r;
        static_cast<ScoreMod &>(r) = m;
        r.codes = entries_are_keys ? b->codes_in : b->codes_out;
        r.table = b->table;
        r.ds = b->ds;
        return r;
    } else {
        return m;
    }
}

// f(DROP, BIAS, SP) with compile-time values
template <bool BUCKETS, typename F> void pick(bool drop, bool biased, int parts, F &&f) {
    using std::integral_constant;
    auto with_parts = [&](auto d, auto b) {
        if (parts == 4) f(d, b, integral_constant<int, 4>{});
        else if (parts == 2) f(d, b, integral_constant<int, 2>{});
        else f(d, b, integral_constant<int, 1>{});
    };
    auto with_bias = [&](auto d) {
        if (!BUCKETS && biased) with_parts(d, integral_constant<int, BUCKETS ? 0 : 1>{});
        else with_parts(d, integral_constant<int, 0>{});
    };
    if (drop) with_bias(integral_constant<bool, true>{});
    else with_bias(integral_constant<bool, false>{});
}

template <typename T, int H, bool BUCKETS = false>
int run_forward(const bpt_plan *P, const bpt_score *sc, const void *q, const void *k, const void *v, const float *bias, void *o, float *lse, void *ws,
                float scale, Dropout drop, hipStream_t s, const BucketArgs *buckets = nullptr) {
    constexpr int D = 64, HW = 4;
    float *ws_acc = (float *)ws, *ws_ml = ws_acc ? ws_acc + (size_t)P->n_slots * H * D : nullptr;
    const auto md = with_buckets<BUCKETS>(make_mod(sc, scale, true, nullptr), buckets, true);
    if (P->n_groups == 0) {
        auto rows = [&](auto nw) {
            hipLaunchKernelGGL((k_score_fwd_rows<T, H, D, FAST_BATCH, nw(), BUCKETS>), dim3(nw() == 1 ? grid_for(P) : (int)P->n_items), dim3(nw() == 1 ? BLOCK : nw() * WAVE), 0,
                               s, *P, (const T *)q, (const T *)k, (const T *)v, (T *)o, lse, ws_acc, ws_ml, scale * LOG2E, md);
        };
        switch (row_parts(P, H * D)) {
        case 8: rows(std::integral_constant<int, 8>{}); break;
        case 4: rows(std::integral_constant<int, 4>{}); break;
        default: rows(std::integral_constant<int, 1>{}); break;
        }
    } else
    pick<BUCKETS>(drop.thr != 0, bias != nullptr, tile_parts(P, H, sizeof(T)), [&](auto dr, auto bi, auto sp) {
        const dim3 grid((unsigned)(group_grid(P) * (H * sp() / HW))), block(HW * WAVE);
        if constexpr (sizeof(T) == 4)
            hipLaunchKernelGGL((k_attn_fwd_tile<T, H, D, HW, dr(), bi(), false, sp(), true, BUCKETS>), grid, block, 0, s, *P, (const T *)q, (const T *)k, (const T *)v,
                               (T *)o, lse, ws_acc, ws_ml, scale * LOG2E, drop.thr, drop.seed, drop.inv, bias, Narrow{}, Keep{}, md);
        else
            hipLaunchKernelGGL((k_attn_fwd_rows_bf16<H, D, HW, TILE_BF16_WPE, dr(), bi(), sp(), true, BUCKETS>), grid, block, 0, s, *P, (const T *)q, (const T *)k,
                               (const T *)v, (T *)o, lse, ws_acc, ws_ml, scale * LOG2E, drop.thr, drop.seed, drop.inv, bias, md);
    });
    const int st = launch_status();
    if (st != BPT_OK || P->n_heavy == 0) return st;
    hipLaunchKernelGGL((k_attn_fwd_combine<T, H, D, false, true>), dim3((unsigned)P->n_heavy, H * D / WAVE), dim3(BLOCK), 0, s, P->heavy, (const float *)ws_acc,
                       (const float *)ws_ml, (T *)o, lse, Narrow{}, (T *)nullptr);
    return launch_status();
}

template <typename T, int H, bool BUCKETS = false>
int run_backward(const bpt_plan *Pin, const bpt_plan *Pout, const bpt_score *sc, const void *q, const void *k, const void *v, const float *bias, const void *o,
                 const void *d_o, const float *lse, void *dq, void *dk, void *dv, float *ds_out, float *dslopes, void *ws, float scale, Dropout drop,
                 hipStream_t s, const BucketArgs *buckets = nullptr) {
    constexpr int D = 64, HW = 4;
    const int dtype = sizeof(T) == 4 ? BPT_F32 : BPT_BF16;
    const bool biased = bias != nullptr, again = sizeof(T) == 2 && !biased;      // (bfloat16 forms (p, ds) again as the layer without options does)
    char *at = (char *)ws;
    void *scratch = at;
    at += scratch_bytes(Pin, Pout, H, dtype, biased);
    float *part = dslopes ? (float *)at : nullptr;
    at += slope_bytes(Pin, H);
    const SplitSums split = split_sums(at, Pin, H, again);
    at += split_bytes(Pin, H, again);
    float *ws_dq = (float *)at, *ws_dk = ws_dq + (size_t)Pin->n_slots * H * D, *ws_dv = ws_dk + (size_t)Pout->n_slots * H * D;
    const int parts_in = tile_parts(Pin, H, sizeof(T)), parts_out = tile_parts(Pout, H, sizeof(T));
    auto md = with_buckets<BUCKETS>(make_mod(sc, scale, true, part), buckets, true);
    const bool fixed = split_counts(Pin, again, dslopes != nullptr, sizeof(T) == 2);
    md.split = fixed ? split.sums : nullptr;
    md.low = split.low;
    pick<BUCKETS>(drop.thr != 0, biased, parts_in, [&](auto dr, auto bi, auto sp) {
        const dim3 grid((unsigned)(group_grid(Pin) * (H * sp() / HW))), block(HW * WAVE);
        if constexpr (sizeof(T) == 4)
            hipLaunchKernelGGL((k_attn_bwd_dst_tile<T, H, D, HW, dr(), bi(), false, sp(), true, BUCKETS>), grid, block, 0, s, *Pin, (const T *)q, (const T *)k, (const T *)v,
                               (const T *)o, (const T *)d_o, lse, (T *)dq, (float2 *)scratch, ws_dq, scale, scale * LOG2E, drop.thr, drop.seed, drop.inv, bias,
                               ds_out, Narrow{}, md);
        else
            hipLaunchKernelGGL((k_attn_bwd_dst_rows_bf16<H, D, HW, TILE_BF16_WPE_DST, dr(), bi(), bi() != 0, sp(), true, BUCKETS>), grid, block, 0, s, *Pin, (const T *)q,
                               (const T *)k, (const T *)v, (const T *)o, (const T *)d_o, lse, (T *)dq, (uint32_t *)scratch, (float2 *)scratch, ws_dq, scale,
                               scale * LOG2E, drop.thr, drop.seed, drop.inv, bias, ds_out, md);
    });
    int st = launch_status();
    if (st != BPT_OK) return st;
    if (fixed)
        hipLaunchKernelGGL(k_score_split, dim3((unsigned)Pin->n_heavy), dim3(BLOCK), 0, s, Pin->heavy, (const float4 *)split.sums,
                           again ? (float2 *)scratch : (float2 *)nullptr, split.fix, H);
    pick<BUCKETS>(drop.thr != 0, biased, parts_out, [&](auto dr, auto bi, auto sp) {
        const dim3 grid((unsigned)(group_grid(Pout) * (H * sp() / HW))), block(HW * WAVE);
        if constexpr (sizeof(T) == 4)
            hipLaunchKernelGGL((k_attn_bwd_src_tile<T, H, D, HW, false, sp(), true>), grid, block, 0, s, *Pout, (const T *)q, (const T *)d_o, (const float2 *)scratch,
                               (T *)dk, (T *)dv, ws_dk, ws_dv, Narrow{});
        else if constexpr (bi() != 0)
            hipLaunchKernelGGL((k_attn_bwd_src_tile_bf16<H, D, HW, TILE_BF16_WPE_SRC, false, sp(), true>), grid, block, 0, s, *Pout, (const T *)q, (const T *)d_o,
                               (const uint32_t *)scratch, (T *)dk, (T *)dv, ws_dk, ws_dv, Narrow{});
        else
            hipLaunchKernelGGL((k_attn_bwd_src_tile_bf16_again<H, D, HW, TILE_BF16_WPE_AGAIN, dr(), sp(), true, BUCKETS>), grid, block, 0, s, *Pout, (const T *)q,
                               (const T *)k, (const T *)v, (const T *)d_o, (const float2 *)scratch, (T *)dk, (T *)dv, ws_dk, ws_dv, scale, scale * LOG2E,
                               drop.thr, drop.seed, drop.inv, with_buckets<BUCKETS>(make_mod(sc, scale, false, nullptr), buckets, false));
    });
    st = launch_status();
    if (st != BPT_OK) return st;
    const SlopeSum sum{part, Pin->grp_chunks + 8, H, parts_in, split.fix, fixed ? (int)Pin->n_heavy : 0, dslopes ? H : 0, dslopes};
    return run_merge<T, false>(sum, Pin, Pout, ws_dq, again && fixed ? split.low : nullptr, (T *)dq, ws_dk, (T *)dk, (T *)dv, H * D, Narrow{}, s);
}

// Heads of fewer than 64 columns, read as they are.
template <typename T>
int run_forward_narrow(const bpt_plan *P, const bpt_score *sc, const void *q, const void *k, const void *v, void *o, float *lse, void *ws, float scale,
                       Dropout drop, const Narrow &nw, hipStream_t s) {
    float *ws_acc = (float *)ws, *ws_ml = ws_acc ? ws_acc + (size_t)P->n_slots * nw.h * 64 : nullptr;
    const ScoreMod md = make_mod(sc, scale, true, nullptr);
    const int parts = tile_parts(P, nw.heads, sizeof(T));
    const Narrow np = narrow_parts(nw, parts);
    pick<false>(drop.thr != 0, false, parts, [&](auto dr, auto, auto sp) {
        constexpr int HW = sp() == 1 ? NARROW_HW : sp();
        const dim3 grid((unsigned)(group_grid(P) * np.slices)), block(HW * WAVE);
        if constexpr (sizeof(T) == 4)
            hipLaunchKernelGGL((k_attn_fwd_tile<T, 16, 64, HW, dr(), 0, true, sp(), true>), grid, block, 0, s, *P, (const T *)q, (const T *)k, (const T *)v, (T *)o,
                               lse, ws_acc, ws_ml, scale * LOG2E, drop.thr, drop.seed, drop.inv, (const float *)nullptr, np, Keep{}, md);
        else
            hipLaunchKernelGGL((k_attn_fwd_tile_bf16<16, 64, HW, TILE_BF16_WPE, dr(), sp(), true>), grid, block, 0, s, *P, (const T *)q, (const T *)k, (const T *)v,
                               (T *)o, lse, ws_acc, ws_ml, scale * LOG2E, drop.thr, drop.seed, drop.inv, np, Keep{}, md);
    });
    const int st = launch_status();
    if (st != BPT_OK || P->n_heavy == 0) return st;
    hipLaunchKernelGGL((k_attn_fwd_combine<T, 16, 64, true, true>), dim3((unsigned)P->n_heavy, nw.heads), dim3(BLOCK), 0, s, P->heavy, (const float *)ws_acc,
                       (const float *)ws_ml, (T *)o, lse, nw, (T *)nullptr);
    return launch_status();
}

template <typename T>
int run_backward_narrow(const bpt_plan *Pin, const bpt_plan *Pout, const bpt_score *sc, const void *q_, const void *k_, const void *v_, const void *o_,
                        const void *d_o_, const float *lse, void *dq_, void *dk_, void *dv_, float *dslopes, void *ws, float scale, Dropout drop, const Narrow &nw,
                        hipStream_t s) {
    constexpr bool F32 = sizeof(T) == 4;
    const T *q = (const T *)q_, *k = (const T *)k_, *v = (const T *)v_, *o = (const T *)o_, *d_o = (const T *)d_o_;
    T *dq = (T *)dq_, *dk = (T *)dk_, *dv = (T *)dv_;
    char *at = (char *)ws;
    float2 *scratch = (float2 *)at;
    at += scratch_bytes(Pin, Pout, nw.h, F32 ? BPT_F32 : BPT_BF16, false);
    float *part = dslopes ? (float *)at : nullptr;
    at += slope_bytes(Pin, nw.h);
    const SplitSums split = split_sums(at, Pin, nw.h, !F32);
    at += split_bytes(Pin, nw.h, !F32);
    const int C = nw.h * 64;
    float *ws_dq = (float *)at, *ws_dk = ws_dq + (size_t)Pin->n_slots * C, *ws_dv = ws_dk + (size_t)Pout->n_slots * C;
    const int parts = tile_parts(Pin, nw.heads, sizeof(T)), parts_src = tile_parts(Pout, nw.heads, sizeof(T));
    const Narrow np = narrow_parts(nw, parts), np_src = narrow_parts(nw, parts_src);
    ScoreMod md = make_mod(sc, scale, true, part);
    const bool fixed = split_counts(Pin, !F32, dslopes != nullptr, !F32);
    md.split = fixed ? split.sums : nullptr;
    md.low = split.low;
    pick<false>(drop.thr != 0, false, parts, [&](auto dr, auto, auto sp) {
        constexpr int HW = sp() == 1 ? NARROW_HW : sp();
        const dim3 grid((unsigned)(group_grid(Pin) * np.slices)), block(HW * WAVE);
        if constexpr (F32)
            hipLaunchKernelGGL((k_attn_bwd_dst_tile<float, 16, 64, HW, dr(), 0, true, sp(), true>), grid, block, 0, s, *Pin, q, k, v, o, d_o, lse, dq, scratch, ws_dq,
                               scale, scale * LOG2E, drop.thr, drop.seed, drop.inv, (const float *)nullptr, (float *)nullptr, np, md);
        else
            hipLaunchKernelGGL((k_score_bwd_dst_narrow_bf16<HW, dr(), sp()>), grid, block, 0, s, *Pin, q, k, v, o, d_o, lse, dq, scratch, ws_dq, scale, scale * LOG2E,
                               drop.thr, drop.seed, drop.inv, np, md);
    });
    int st = launch_status();
    if (st != BPT_OK) return st;
    if (fixed)          // (the padding heads' sums are not used)
        hipLaunchKernelGGL(k_score_split, dim3((unsigned)Pin->n_heavy), dim3(BLOCK), 0, s, Pin->heavy, (const float4 *)split.sums, F32 ? nullptr : scratch, split.fix, nw.h);
    pick<false>(!F32 && drop.thr != 0, false, parts_src, [&](auto dr, auto, auto sp) {
        constexpr int HW = sp() == 1 ? NARROW_HW : sp();
        const dim3 grid((unsigned)(group_grid(Pout) * np_src.slices)), block(HW * WAVE);
        if constexpr (F32)
            hipLaunchKernelGGL((k_attn_bwd_src_tile<float, 16, 64, HW, true, sp(), true>), grid, block, 0, s, *Pout, q, d_o, (const float2 *)scratch, dk, dv, ws_dk, ws_dv,
                               np_src);
        else
            hipLaunchKernelGGL((k_score_bwd_src_narrow_bf16<HW, dr(), sp()>), grid, block, 0, s, *Pout, q, k, v, d_o, (const float2 *)scratch, dk, dv, ws_dk, ws_dv,
                               scale, scale * LOG2E, drop.thr, drop.seed, drop.inv, np_src, make_mod(sc, scale, false, nullptr));
    });
    st = launch_status();
    if (st != BPT_OK) return st;
    const SlopeSum sum{part, Pin->grp_chunks + 8, nw.h, parts, split.fix, fixed ? (int)Pin->n_heavy : 0, dslopes ? nw.heads : 0, dslopes};
    return run_merge<T, true>(sum, Pin, Pout, ws_dq, !F32 && fixed ? split.low : nullptr, dq, ws_dk, dk, dv, C, nw, s);
}

inline int check_score(const bpt_plan *P, const bpt_score *sc, int heads, int d, int h, int dtype, float scale, float dropout_p, const float *bias,
                       Narrow &nw, bool forward) {
    const int st = check_plan(P, true);
    if (st != BPT_OK) return st;
    if (!sc) return BPT_ERR_NULL;
    if (dtype != BPT_F32 && dtype != BPT_BF16) return dtype == BPT_F64 ? BPT_ERR_UNSUPPORTED : BPT_ERR_DTYPE;
    if (h != 8 && h != 16 && !(h == 4 && dtype == BPT_F32)) return BPT_ERR_UNSUPPORTED;
    if (heads < 1 || d < 1) return BPT_ERR_SHAPE;
    const bool narrow = heads != h || d != 64;
    if (narrow && ((dtype != BPT_F32 && d % 2 != 0) || bias || heads > h || d < 4 || d > 64)) return BPT_ERR_UNSUPPORTED;
    nw = narrow ? Narrow{d, heads, h, (heads + NARROW_HW - 1) / NARROW_HW} : Narrow{};
    // (within these bounds the polynomial's coefficients and squares of scores are ordinary numbers: make_mod, tile_mod_scores)
    const bool capped = sc->cap != 0.f;
    if (capped && !(sc->cap >= 0.9e-10f && sc->cap <= 1.1e10f && fabsf(scale) <= 1.01e4f * sc->cap && fabsf(scale) <= 1.01e6f)) return BPT_ERR_SIZE;
    if (!(dropout_p >= 0.f && dropout_p < 1.f)) return BPT_ERR_SIZE;
    if (sc->slopes && (!sc->pos_q || !sc->pos_k)) return BPT_ERR_NULL;
    if (P->n_rows == 0) return P->n_edges == 0 ? BPT_OK : BPT_ERR_UNSUPPORTED;
    if (forward && P->n_groups == 0 && !narrow && !bias && !(dropout_p > 0.f)) return BPT_OK;
    if (!has_tiles(P, h, 64, dtype == BPT_BF16 ? 2 : 4)) return BPT_ERR_UNSUPPORTED;
    if ((bias || dropout_p > 0.f || narrow) && !P->grp_eids) return BPT_ERR_PLAN;
    if (bias && P->bias_by_pair) return BPT_ERR_PLAN;
    return BPT_OK;
}
inline bool on16(std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (!aligned16(p)) return false;
    return true;
}
inline bool on4(std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (reinterpret_cast<uintptr_t>(p) & 3) return false;
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
