// libbptbias: gfx950 kernels of a learned bias of attention scores by buckets, and its gradient: the separate operator, and the fused attention, whose tile kernels
// (bpttiles.h) have BUCKETS forms (C ABI in include/bptbias.h).
#include "bptmod.h"

#include "../../include/bptbias.h"

namespace {

// ---- the term by edge id -----------------------------------------------------------------------------------------------------------
// For the separate operator, and tables of more buckets than a byte counts.  bias[e][head] = table[buckets[e]][head] factor: 8 bytes an edge read and h values written, the table comes
// from the caches.  A thread has one value, so the division and the loads of each bound it, not memory (8.4 million edges of 16 heads, 64 buckets: float32 333 us, 1.8 TB/s; bfloat16 303).
template <typename T, typename O>
__global__ __launch_bounds__(BLOCK) void k_bucket_rows(const T *__restrict__ table, const int64_t *__restrict__ buckets, O *__restrict__ bias, int64_t n_edges,
                                                       int64_t n_buckets, int h, typename Elem<T>::acc_t factor, int spare_row) {
    using A = typename Elem<T>::acc_t;
    const int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * BLOCK + threadIdx.x, e = i / h;
    const int head = (int)(i - e * h);
    if (e >= n_edges + spare_row) return;
    const int64_t b = e < n_edges ? buckets[e] : -1;
    Elem<O>::st(bias + i, (uint64_t)b < (uint64_t)n_buckets ? (A)Elem<T>::ld(table + b * h + head) * factor : A(0));
}

// ---- its gradient --------------------------------------------------------------------------------------------------------------------
// dtable[b][head] = factor sum over the edges of bucket b of ds[e][head].  A lane owns a column of
// sums in LDS, one a bucket, so nobody shares an address and the order of every sum is fixed: lanes of one head, wavefronts, workgroups
// in theirs.  64 / h edges a wavefront and step (of more than 64 heads, 64 by 64).
// Up to SUMS_WIDE buckets a workgroup of four wavefronts has them all (64 KB at 64); of more, one wavefront has 256 and the
// edges are walked once for each 256.  Bound by LDS, where a sum is read and written for every value, one after another, by two workgroups a compute unit (8.4 million edges of 16 heads,
// with the launch behind: 64 buckets float32 598 us, 1.0 TB/s, bfloat16 817; 256 buckets, a wavefront a workgroup, 2147 and 2514, 1000 buckets 8426 and 10150).
constexpr int SUMS_WIDE = 64, SUMS_LONG = 256;
template <typename D, typename A, int WAVES, int ROOM>
__global__ __launch_bounds__(WAVES *WAVE) void k_bucket_sums(const D *__restrict__ ds, const int64_t *__restrict__ buckets, A *__restrict__ part, int64_t n_edges,
                                                             int64_t n_buckets, int h) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    A *const sums = reinterpret_cast<A *>(lds) + (size_t)(threadIdx.x >> 6) * ROOM * WAVE;
    const int lane = threadIdx.x & 63, h0 = (int)blockIdx.y * WAVE, heads = min(h - h0, WAVE), per = WAVE / heads, mine = lane / heads;
    const int64_t b0 = (int64_t)blockIdx.z * ROOM;
    const int room = (int)min((int64_t)ROOM, n_buckets - b0);
    for (int b = 0; b < room; ++b) sums[b * WAVE + lane] = A(0);
    constexpr int U = 8;
    const int64_t wave = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * WAVES;
    if (mine < per) {
        for (int64_t e0 = wave * per * U; e0 < n_edges; e0 += waves * per * U) {
            int64_t b[U];
            A x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t e = e0 + u * per + mine;
                b[u] = e < n_edges ? buckets[e] - b0 : -1;
                x[u] = e < n_edges ? (A)Elem<D>::ld(ds + e * h + h0 + lane % heads) : A(0);
            }
            issue_loads_first();
#pragma unroll
            for (int u = 0; u < U; ++u)
                if ((uint64_t)b[u] < (uint64_t)room) sums[(int)b[u] * WAVE + lane] += x[u];
        }
    }
    __syncthreads();
    const A *const all = reinterpret_cast<const A *>(lds);
    for (int i = threadIdx.x; i < room * heads; i += WAVES * WAVE) {
        const int b = i / heads, head = i - b * heads;
        A v = A(0);
        for (int w = 0; w < WAVES; ++w)
            for (int m = 0; m < per; ++m) v += all[((size_t)w * ROOM + b) * WAVE + m * heads + head];
        part[((int64_t)blockIdx.x * n_buckets + b0 + b) * h + h0 + head] = v;
    }
}
// sixteen lanes an element take parts p, p + 16, ...; the sixteen are added in their order
template <typename T, typename A>
__global__ __launch_bounds__(BLOCK) void k_bucket_finish(const A *__restrict__ part, int parts, T *__restrict__ dtable, int64_t n, A factor) {
    __shared__ A meet[16][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int64_t at = (int64_t)blockIdx.x * 16 + c;
    A v = A(0);
    if (at < n)
        for (int p = k; p < parts; p += 16) v += part[(int64_t)p * n + at];
    meet[k][c] = v;
    __syncthreads();
    if (k != 0 || at >= n) return;
    v = meet[0][c];
#pragma unroll
    for (int i = 1; i < 16; ++i) v += meet[i][c];
    Elem<T>::st(dtable + at, v * factor);
}

constexpr int SUMS_PARTS = 512;
// workgroups that share the edges: each has 64 steps of them at least
inline int sums_parts(int64_t n_edges, int h) {
    const int64_t per = std::max(1, WAVE / std::min(h, WAVE));
    return (int)std::max<int64_t>(1, std::min<int64_t>(SUMS_PARTS, n_edges / (per * 64) + 1));
}

template <typename T, typename O>
int run_rows(const void *table, const int64_t *buckets, void *bias, int64_t n_edges, int64_t n_buckets, int h, double factor, int spare, hipStream_t s) {
    // (an axis of a launch counts its threads in 32 bits)
    const int64_t blocks = ((n_edges + spare) * h + BLOCK - 1) / BLOCK, along = std::min<int64_t>(blocks, (int64_t)1 << 23);
    hipLaunchKernelGGL((k_bucket_rows<T, O>), dim3((unsigned)along, (unsigned)((blocks + along - 1) / along)), dim3(BLOCK), 0, s, (const T *)table, buckets, (O *)bias, n_edges,
                       n_buckets, h, (typename Elem<T>::acc_t)factor, spare);
    return launch_status();
}
template <typename D, typename T>
int run_sums(const void *ds, const int64_t *buckets, void *dtable, void *ws, int64_t n_edges, int64_t n_buckets, int h, double factor, hipStream_t s) {
    using A = typename Elem<D>::acc_t;
    const int parts = sums_parts(n_edges, h);
    const unsigned chunks = (unsigned)((h + WAVE - 1) / WAVE);
    constexpr int WIDE = SUMS_WIDE * 4 / (int)sizeof(A), LONG = SUMS_LONG * 4 / (int)sizeof(A);
    if (n_buckets <= WIDE)
        hipLaunchKernelGGL((k_bucket_sums<D, A, 4, WIDE>), dim3(parts, chunks, 1), dim3(4 * WAVE), 4 * WIDE * WAVE * sizeof(A), s, (const D *)ds, buckets, (A *)ws, n_edges,
                           n_buckets, h);
    else
        hipLaunchKernelGGL((k_bucket_sums<D, A, 1, LONG>), dim3(parts, chunks, (unsigned)((n_buckets + LONG - 1) / LONG)), dim3(WAVE), LONG * WAVE * sizeof(A), s,
                           (const D *)ds, buckets, (A *)ws, n_edges, n_buckets, h);
    const int st = launch_status();
    if (st != BPT_OK) return st;
    hipLaunchKernelGGL((k_bucket_finish<T, A>), dim3((unsigned)((n_buckets * h + 15) / 16)), dim3(BLOCK), 0, s, (const A *)ws, parts, (T *)dtable, n_buckets * h, (A)factor);
    return launch_status();
}

// ---- the fused attention -----------------------------------------------------------------------------------------------------------
// One byte a place says which of a head's biases a pair takes, so the passes read 1 / (4 h) of what the term itself would be (float32, h heads, each way), and nothing
// of an edge's size is written but ds, which is summed up by buckets behind the backward: in float32 from the scratch that the sides hand over anyway, in bfloat16, whose
// sides hand over none, from the source side's own, in 32 bits: L = 32768, k = 8, 16 heads, 211 MB each way.  (In bfloat16 the sums of a table whose terms cancel came out
// 1.5 times as far off as their own rounding.)
inline int64_t places(const bpt_plan *p) { return p->n_groups > 0 ? p->n_grp_entries * TILE_R : p->n_edges; }
inline const int32_t *place_eids(const bpt_plan *p) { return p->n_groups > 0 ? p->grp_eids : p->eid; }
inline int64_t table_bytes(int h) { return (int64_t)h * 256 * 4; }
struct Prepared {
    float *table;
    uint8_t *codes_in, *codes_pairs, *codes_out;      // (the last two for a backward: by pair numbers of the side whose ds is summed up, and by places)
    Prepared(void *at, const bpt_plan *in, int h)
        : table((float *)at), codes_in((uint8_t *)at + table_bytes(h)), codes_pairs(codes_in + round16(places(in))), codes_out(codes_pairs + round16(in->n_edges)) {}
};

// What a table's value of -HIDES and below stands for is -infinity.  A score of that size and a row's lse are off by 3 percent of a factor, of one of 10^9 by any: rows of nothing
// but such masks would have probabilities that do not add up, and one of the type's lowest values divided by the scale is no number any more.
constexpr float HIDES = BPT_HIDES;
// Bound by memory: the edge ids of either side's places, and a bucket of 8 bytes for each that exists, from the caches (L = 8192 6 us; L = 32768, k = 8 36 us).
// blockIdx.y: 0 the tables, 1 and 2 the places of either side, four a thread; by_pair: the side whose pairs' codes are wanted too, or 0
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_bucket_prepare(const T *__restrict__ table, const int64_t *__restrict__ buckets, int n_buckets, int heads, int h, float factor,
                                                          int64_t n_edges, const int32_t *__restrict__ eids_in, int64_t n_in, const int32_t *__restrict__ eids_out,
                                                          int64_t n_out, float *__restrict__ tables, uint8_t *__restrict__ codes_in, uint8_t *__restrict__ codes_out,
                                                          const int4 *__restrict__ entries, int by_pair, uint8_t *__restrict__ codes_pairs) {
    const int64_t first = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) * 4;
    if (blockIdx.y == 0) {
        for (int64_t i = first; i < first + 4 && i < (int64_t)h * 256; ++i) {
            const int head = (int)(i >> 8), b = (int)i & 255;
            const float x = head < heads && b < n_buckets ? Elem<T>::ld(table + (int64_t)b * heads + head) : 0.f;
            tables[i] = (x <= -HIDES ? -INFINITY : x) * factor;
        }
        return;
    }
    const int32_t *const eids = blockIdx.y == 1 ? eids_in : eids_out;
    uint8_t *const codes = blockIdx.y == 1 ? codes_in : codes_out;
    const int64_t n = blockIdx.y == 1 ? n_in : n_out;
    int64_t e[4], b[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) e[u] = first + u < n ? eids[first + u] : -1;
#pragma unroll
    for (int u = 0; u < 4; ++u) b[u] = (uint64_t)e[u] < (uint64_t)n_edges ? buckets[e[u]] : -1;
    uint32_t word = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) word |= ((uint64_t)b[u] < (uint64_t)n_buckets ? (uint32_t)b[u] : (uint32_t)NO_BUCKET) << 8 * u;
    if (by_pair == (int)blockIdx.y && first < n) {                // (four places are of one entry)
        const int4 en = entries[first / TILE_R];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int m = (int)(first % TILE_R) + u;
            const int64_t pair = tile_pair_number(en.z, en.y, m);
            if (((en.y >> m) & 1) && (uint64_t)pair < (uint64_t)n_edges) codes_pairs[pair] = (uint8_t)(word >> 8 * u);
        }
    }
    if (first + 4 <= n) {
        *reinterpret_cast<uint32_t *>(codes + first) = word;
    } else {
        for (int u = 0; u < 4; ++u)
            if (first + u < n) codes[first + u] = (uint8_t)(word >> 8 * u);
    }
}

// dtable's parts from ds by pairs, [head][pair]: a workgroup has one head, a lane four pairs at a time and a column of sums in LDS, as k_bucket_sums.
// float32: ds is the second of the pairs' (p, ds); bfloat16: the source side's own.  Bound by memory: L = 32768, k = 8, 16 heads 51 us (264 MB, 5.2 TB/s), L = 8192, 8 heads
// float32 7 us.  By places, the entries read beside them and a load of one element a lane, those were 505 and 23 us.
template <typename T> struct PairDs { typedef float2 type; };
template <> struct PairDs<bf16_t> { typedef float type; };
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES *WAVE) void k_bucket_pairs(const uint8_t *__restrict__ codes, const typename PairDs<T>::type *__restrict__ ds, int64_t n, int room,
                                                              float *__restrict__ part, int heads) {
    constexpr int U = sizeof(T) == 4 ? 2 : 4;
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
    extern __shared__ __attribute__((aligned(16))) char lds[];
    float *const sums = reinterpret_cast<float *>(lds) + (threadIdx.x >> 6) * room * WAVE;
    const int lane = threadIdx.x & 63, head = (int)blockIdx.y;
    for (int b = 0; b < room; ++b) sums[b * WAVE + lane] = 0.f;
    const float *const ds_h = reinterpret_cast<const float *>(ds + (int64_t)head * n);
    const int64_t wave = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * WAVES, whole = n & ~3;
    for (int64_t i0 = wave * WAVE * 4 * U; i0 < whole; i0 += waves * WAVE * 4 * U) {
        uint32_t word[U];
        float4u x[U], y[sizeof(T) == 4 ? U : 1];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = i0 + (u * WAVE + lane) * 4, at = min(i, whole - 4);
            word[u] = *reinterpret_cast<const uint32_t *>(codes + at);
            if (i >= whole) word[u] = 0xFFFFFFFFu;
            if constexpr (sizeof(T) == 4) {
                x[u] = *reinterpret_cast<const float4u *>(ds_h + 2 * at);
                y[u] = *reinterpret_cast<const float4u *>(ds_h + 2 * at + 4);
            } else {
                x[u] = *reinterpret_cast<const float4u *>(ds_h + at);
            }
        }
        issue_loads_first();
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = (int)(word[u] >> 8 * j) & 255;
                float v;
                if constexpr (sizeof(T) == 4) v = j < 2 ? x[u][2 * (j & 1) + 1] : y[u][2 * (j & 1) + 1];
                else v = x[u][j];
                if (b < room) sums[b * WAVE + lane] += v;
            }
        }
    }
    if (blockIdx.x == 0 && (int)threadIdx.x < (int)(n - whole)) {      // (up to three behind the last four)
        const int64_t i = whole + threadIdx.x;
        const int b = codes[i];
        if (b < room) sums[b * WAVE + lane] += ds_h[sizeof(T) == 4 ? 2 * i + 1 : i];
    }
    __syncthreads();
    const float *const all = reinterpret_cast<const float *>(lds);
    // a bucket a quarter of a wavefront: sixteen lanes add four columns of every wavefront's each, and meet in a fixed order
    for (int b0 = 0; b0 < room; b0 += WAVES * 4) {
        const int b = b0 + (int)threadIdx.x / 16, c = threadIdx.x & 15;
        float v = 0.f;
        if (b < room) {
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
#pragma unroll
                for (int u = 0; u < 4; ++u) v += all[((size_t)w * room + b) * WAVE + 16 * u + c];
        }
        v = head_sum<16>(v);
        if (b < room && c == 0) part[((int64_t)blockIdx.x * room + b) * heads + head] = v;
    }
}

// as many workgroups as stay on the chip at a time, of at least a turn's pairs each
constexpr int PAIR_PARTS = 256;
template <typename T>
int run_pairs(int64_t n, const uint8_t *codes, const typename PairDs<T>::type *ds, float *part, T *dtable, int n_buckets, int heads, float factor, hipStream_t s) {
    const int waves = n_buckets <= SUMS_WIDE ? 4 : 1, most = std::min(PAIR_PARTS, (1024 + heads - 1) / heads);
    const int parts = (int)std::min<int64_t>(most, n / (512 * waves) + 1);
    const dim3 grid((unsigned)parts, (unsigned)heads);
    const size_t bytes = (size_t)waves * n_buckets * WAVE * 4;
    if (waves == 4) hipLaunchKernelGGL((k_bucket_pairs<T, 4>), grid, dim3(4 * WAVE), bytes, s, codes, ds, n, n_buckets, part, heads);
    else hipLaunchKernelGGL((k_bucket_pairs<T, 1>), grid, dim3(WAVE), bytes, s, codes, ds, n, n_buckets, part, heads);
    const int st = launch_status();
    if (st != BPT_OK) return st;
    hipLaunchKernelGGL((k_bucket_finish<T, float>), dim3((unsigned)(((int64_t)n_buckets * heads + 15) / 16)), dim3(BLOCK), 0, s, part, parts, dtable,
                       (int64_t)n_buckets * heads, factor);
    return launch_status();
}

inline int64_t attention_bytes(const bpt_plan *in, const bpt_plan *out, int h, int dtype) {
    return scratch_bytes(in, out, h, dtype, false) + slope_bytes(in, h) + split_bytes(in, h, dtype == BPT_BF16) + round16((in->n_slots + 2 * out->n_slots) * (int64_t)h * 64 * 4);
}
inline int64_t ds_bytes(const bpt_plan *out, int h, int dtype) { return dtype == BPT_BF16 ? round16(out->n_edges * h * 4) : 0; }

inline bool is_type(int dtype) { return dtype == BPT_F32 || dtype == BPT_F64 || dtype == BPT_BF16; }
inline bool is_size(int64_t n_edges, int64_t n_buckets, int h) {
    return n_edges >= 0 && n_edges <= (int64_t)1 << 31 && n_buckets >= 1 && n_buckets <= 65536 && h >= 1 && h <= 1024 && (n_edges + 1) * h <= (int64_t)1 << 38;
}

}  // namespace

extern "C" {

int bpt_bucket_bias_forward(const void *table, const int64_t *buckets, void *bias, int64_t n_edges, int64_t n_buckets, int h, double factor, int spare_row, int dtype,
                            int out_dtype, void *stream) {
    if (!is_type(dtype) || !(out_dtype == dtype || (dtype == BPT_BF16 && out_dtype == BPT_F32))) return BPT_ERR_DTYPE;
    if (!is_size(n_edges, n_buckets, h) || (spare_row != 0 && spare_row != 1)) return BPT_ERR_SIZE;
    if (n_edges + spare_row == 0) return BPT_OK;
    if (!table || !bias || (n_edges > 0 && !buckets)) return BPT_ERR_NULL;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == BPT_F64) return run_rows<double, double>(table, buckets, bias, n_edges, n_buckets, h, factor, spare_row, s);
    if (dtype == BPT_F32) return run_rows<float, float>(table, buckets, bias, n_edges, n_buckets, h, factor, spare_row, s);
    if (out_dtype == BPT_F32) return run_rows<bf16_t, float>(table, buckets, bias, n_edges, n_buckets, h, factor, spare_row, s);
    return run_rows<bf16_t, bf16_t>(table, buckets, bias, n_edges, n_buckets, h, factor, spare_row, s);
}

int64_t bpt_bucket_bias_backward_workspace_bytes(int64_t n_edges, int64_t n_buckets, int h, int dtype) {
    if (!is_type(dtype) || !is_size(n_edges, n_buckets, h)) return -1;
    return (int64_t)sums_parts(n_edges, h) * n_buckets * h * (int64_t)acc_size(dtype);
}

int bpt_bucket_bias_backward(const void *ds, const int64_t *buckets, void *dtable, void *workspace, int64_t workspace_bytes, int64_t n_edges, int64_t n_buckets, int h,
                             double factor, int dtype, int ds_dtype, void *stream) {
    if (!is_type(dtype) || !(ds_dtype == dtype || (dtype == BPT_BF16 && ds_dtype == BPT_F32))) return BPT_ERR_DTYPE;
    if (!is_size(n_edges, n_buckets, h)) return BPT_ERR_SIZE;
    if (!dtable || (n_edges > 0 && (!ds || !buckets))) return BPT_ERR_NULL;
    if (!workspace || workspace_bytes < bpt_bucket_bias_backward_workspace_bytes(n_edges, n_buckets, h, dtype) || !aligned16(workspace)) return BPT_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == BPT_F64) return run_sums<double, double>(ds, buckets, dtable, workspace, n_edges, n_buckets, h, factor, s);
    if (dtype == BPT_F32) return run_sums<float, float>(ds, buckets, dtable, workspace, n_edges, n_buckets, h, factor, s);
    if (ds_dtype == BPT_F32) return run_sums<float, bf16_t>(ds, buckets, dtable, workspace, n_edges, n_buckets, h, factor, s);
    return run_sums<bf16_t, bf16_t>(ds, buckets, dtable, workspace, n_edges, n_buckets, h, factor, s);
}

int64_t bpt_bucket_prepare_bytes(const bpt_plan *plan_in, const bpt_plan *plan_out, int h) {
    if (!plan_in || h < 1 || h > 16) return -1;
    return table_bytes(h) + round16(places(plan_in)) + (plan_out ? round16(plan_in->n_edges) + round16(places(plan_out)) : 0);
}

int bpt_bucket_prepare(const bpt_plan *plan_in, const bpt_plan *plan_out, const void *table, const int64_t *buckets, int64_t n_buckets, int heads, int h, float scale,
                       int dtype, void *prepared, void *stream) {
    if (dtype != BPT_F32 && dtype != BPT_BF16) return BPT_ERR_DTYPE;
    if (n_buckets < 1 || n_buckets > BPT_MOST_BUCKETS || heads < 1 || heads > h || h > 16 || !(fabsf(scale) > 0.f && fabsf(scale) < INFINITY)) return BPT_ERR_SIZE;
    for (const bpt_plan *p : {plan_in, plan_out ? plan_out : plan_in}) {
        const int st = check_plan(p, true);
        if (st != BPT_OK) return st;
        if (p->n_groups > 0 && (!p->grp_eids || p->grp_R != TILE_R)) return BPT_ERR_PLAN;
    }
    if (plan_out && (plan_out->n_edges != plan_in->n_edges || plan_in->n_groups == 0 || plan_out->n_groups == 0)) return BPT_ERR_PLAN;
    if (!table || !prepared || (plan_in->n_edges > 0 && !buckets)) return BPT_ERR_NULL;
    if (!aligned16(prepared)) return BPT_ERR_UNSUPPORTED;
    const Prepared pr(prepared, plan_in, h);
    const int64_t in = places(plan_in), out = plan_out ? places(plan_out) : 0, most = std::max<int64_t>(std::max(in, out), h * 256);
    if (most > (((int64_t)1 << 32) - BLOCK) * 4) return BPT_ERR_SIZE;      // (a launch counts its threads in 32 bits)
    const dim3 grid((unsigned)((most + 4 * BLOCK - 1) / (4 * BLOCK)), plan_out ? 3 : 2);
    hipStream_t s = (hipStream_t)stream;
    const int32_t *ei = place_eids(plan_in), *eo = plan_out ? place_eids(plan_out) : nullptr;
    const bpt_plan *const summed = dtype == BPT_F32 ? plan_in : plan_out;
    const int by_pair = plan_out ? (dtype == BPT_F32 ? 1 : 2) : 0;
    const int4 *const entries = plan_out ? (const int4 *)summed->grp_entries : nullptr;
    if (dtype == BPT_F32)
        hipLaunchKernelGGL((k_bucket_prepare<float>), grid, dim3(BLOCK), 0, s, (const float *)table, buckets, (int)n_buckets, heads, h, 1.f / scale, plan_in->n_edges, ei, in,
                           eo, out, pr.table, pr.codes_in, pr.codes_out, entries, by_pair, pr.codes_pairs);
    else
        hipLaunchKernelGGL((k_bucket_prepare<bf16_t>), grid, dim3(BLOCK), 0, s, (const bf16_t *)table, buckets, (int)n_buckets, heads, h, 1.f / scale, plan_in->n_edges, ei,
                           in, eo, out, pr.table, pr.codes_in, pr.codes_out, entries, by_pair, pr.codes_pairs);
    return launch_status();
}

int bpt_bucket_attention_forward(const bpt_plan *plan_in, const bpt_score *score, const void *prepared, const void *q, const void *k, const void *v, void *o, float *lse,
                                 void *workspace, int64_t workspace_bytes, float scale, float dropout_p, uint64_t dropout_seed, int h, int dtype, void *stream) {
    Narrow nw;
    const int st = check_score(plan_in, score, h, 64, h, dtype, scale, dropout_p, nullptr, nw, true);
    if (st != BPT_OK) return st;
    if (plan_in->n_rows == 0) return BPT_OK;
    if (!prepared || !q || !k || !v || !o || !lse) return BPT_ERR_NULL;
    if (plan_in->n_groups > 0 && !plan_in->grp_eids) return BPT_ERR_PLAN;
    if (!aligned16(workspace) || !on16({prepared, q, k, v, o})) return BPT_ERR_UNSUPPORTED;
    const int64_t need = round16(plan_in->n_slots * ((int64_t)h * 64 + 2 * h) * 4);
    if (need > 0 && (!workspace || workspace_bytes < need)) return BPT_ERR_WORKSPACE;
    const Prepared pr(const_cast<void *>(prepared), plan_in, h);
    const BucketArgs b{pr.codes_in, nullptr, pr.table, nullptr};
    const Dropout drop = make_dropout(dropout_p, dropout_seed);
    DISPATCH((run_forward<T, H, true>(plan_in, score, q, k, v, nullptr, o, lse, workspace, scale, drop, (hipStream_t)stream, &b)))
}

int64_t bpt_bucket_attention_backward_workspace_bytes(const bpt_plan *plan_in, const bpt_plan *plan_out, int64_t n_buckets, int heads, int h, int dtype) {
    if (!plan_in || !plan_out || h < 1 || h > 16 || heads < 1 || heads > h || n_buckets < 1 || n_buckets > BPT_MOST_BUCKETS || (dtype != BPT_F32 && dtype != BPT_BF16)) return -1;
    return attention_bytes(plan_in, plan_out, h, dtype) + ds_bytes(plan_out, h, dtype) + (int64_t)PAIR_PARTS * n_buckets * heads * 4;
}

int bpt_bucket_attention_backward(const bpt_plan *plan_in, const bpt_plan *plan_out, const bpt_score *score, const void *prepared, const void *q, const void *k, const void *v,
                                  const void *o, const void *d_o, const float *lse, void *dq, void *dk, void *dv, void *dtable, float *dslopes, void *workspace,
                                  int64_t workspace_bytes, int64_t n_buckets, int heads, float scale, float dropout_p, uint64_t dropout_seed, int h, int dtype,
                                  void *stream) {
    Narrow nw;
    int st = check_score(plan_in, score, h, 64, h, dtype, scale, dropout_p, nullptr, nw, false);
    if (st != BPT_OK) return st;
    st = check_plan(plan_out, true);
    if (st != BPT_OK) return st;
    if (n_buckets < 1 || n_buckets > BPT_MOST_BUCKETS || heads < 1 || heads > h || !(fabsf(scale) > 0.f)) return BPT_ERR_SIZE;
    if (plan_in->n_edges != plan_out->n_edges) return BPT_ERR_PLAN;
    if (plan_in->n_groups == 0 || !has_tiles(plan_out, h, 64, dtype == BPT_BF16 ? 2 : 4) || !plan_out->grp_pairs) return BPT_ERR_UNSUPPORTED;
    if (!plan_in->grp_eids || !plan_out->grp_eids) return BPT_ERR_PLAN;
    if (!prepared || !q || !k || !v || !o || !d_o || !lse || !dq || !dk || !dv || (dslopes && !score->slopes)) return BPT_ERR_NULL;
    if (!aligned16(workspace) || !on16({prepared, q, k, v, o, d_o, dq, dk, dv})) return BPT_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < bpt_bucket_attention_backward_workspace_bytes(plan_in, plan_out, n_buckets, heads, h, dtype)) return BPT_ERR_WORKSPACE;
    const Prepared pr(const_cast<void *>(prepared), plan_in, h);
    char *const behind = (char *)workspace + attention_bytes(plan_in, plan_out, h, dtype);
    const BucketArgs b{pr.codes_in, pr.codes_out, pr.table, dtable && dtype == BPT_BF16 ? (float *)behind : nullptr};
    float *const part = (float *)(behind + ds_bytes(plan_out, h, dtype));
    const Dropout drop = make_dropout(dropout_p, dropout_seed);
    hipStream_t s = (hipStream_t)stream;
    auto attention = [&]() -> int {
        DISPATCH((run_backward<T, H, true>(plan_in, plan_out, score, q, k, v, nullptr, o, d_o, lse, dq, dk, dv, nullptr, dslopes, workspace, scale, drop, s, &b)))
    };
    st = attention();
    if (st != BPT_OK || !dtable) return st;
    if (dtype == BPT_F32)
        return run_pairs<float>(plan_in->n_edges, pr.codes_pairs, (const float2 *)workspace, part, (float *)dtable, n_buckets, heads, 1.f / scale, s);
    return run_pairs<bf16_t>(plan_in->n_edges, pr.codes_pairs, (const float *)behind, part, (bf16_t *)dtable, n_buckets, heads, 1.f / scale, s);
}

}  // extern "C"
