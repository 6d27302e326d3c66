// libbptbias: gfx950 kernels of a learned bias of attention scores by buckets, and its gradient (C ABI in include/bptbias.h).
#include "bpttiles.h"

#include "../../include/bptbias.h"

namespace {

// ---- the term by edge id -----------------------------------------------------------------------------------------------------------
// bias[e][head] = table[buckets[e]][head] factor: bound by memory, 8 bytes an edge read and h values written, the table comes from the caches.
template <typename T, typename O>
__global__ __launch_bounds__(BLOCK) void k_bucket_rows(const T *__restrict__ table, const int64_t *__restrict__ buckets, O *__restrict__ bias, int64_t n_edges,
                                                       int64_t n_buckets, int h, typename Elem<T>::acc_t factor, int spare_row) {
    using A = typename Elem<T>::acc_t;
    const int64_t i = (int64_t)blockIdx.x * BLOCK + threadIdx.x, e = i / h;
    const int head = (int)(i - e * h);
    if (e >= n_edges + spare_row) return;
    const int64_t b = e < n_edges ? buckets[e] : -1;
    Elem<O>::st(bias + i, (uint64_t)b < (uint64_t)n_buckets ? (A)Elem<T>::ld(table + b * h + head) * factor : A(0));
}

// ---- the term in the order of a tile plan's pairs -------------------------------------------------------------------------------
constexpr uint32_t NO_BUCKET = 65535;
__global__ __launch_bounds__(BLOCK) void k_bucket_codes(const int64_t *__restrict__ buckets, const int32_t *__restrict__ eid_of_pair, uint16_t *__restrict__ codes,
                                                        int64_t n_edges, int64_t n_buckets) {
    const int64_t t = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
    if (t >= n_edges) return;
    const int64_t b = buckets[eid_of_pair[t]];
    codes[t] = (uint16_t)((uint64_t)b < (uint64_t)n_buckets ? (uint32_t)b : NO_BUCKET);
}
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_bucket_terms(const T *__restrict__ table, const uint16_t *__restrict__ codes, float *__restrict__ bias, int64_t n_edges, int h,
                                                        float factor) {
    const int64_t t = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
    if (t >= n_edges) return;
    const uint32_t b = codes[t];
    for (int head = 0; head < h; ++head) bias[(int64_t)head * n_edges + t] = b == NO_BUCKET ? 0.f : Elem<T>::ld(table + (int64_t)b * h + head) * factor;
}

// ---- its gradient --------------------------------------------------------------------------------------------------------------------
// dtable[b][head] = factor sum over the edges of bucket b of ds[e][head]: bound by memory, ds and the buckets read once.  A lane owns a column of
// sums in LDS, one a bucket, so nobody shares an address and the order of every sum is fixed: lanes of one head, wavefronts, workgroups
// in theirs.  64 / h edges a wavefront and step (of more than 64 heads, 64 by 64).
// Up to SUMS_WIDE buckets a workgroup of four wavefronts has them all (64 KB at 64); of more, one wavefront has 256 and the
// edges are walked once for each 256.
constexpr int SUMS_WIDE = 64, SUMS_LONG = 256;
// In the order of pairs ds is (h, n_edges): a workgroup has one head, a lane a pair.
template <typename D, typename A, typename B, int WAVES, int ROOM>
__global__ __launch_bounds__(WAVES *WAVE) void k_bucket_sums(const D *__restrict__ ds, const B *__restrict__ buckets, A *__restrict__ part, int64_t n_edges,
                                                             int64_t n_buckets, int h) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    A *const sums = reinterpret_cast<A *>(lds) + (size_t)(threadIdx.x >> 6) * ROOM * WAVE;
    constexpr bool PAIRS = sizeof(B) == 2;
    const int lane = threadIdx.x & 63, h0 = (int)blockIdx.y * (PAIRS ? 1 : WAVE), heads = PAIRS ? 1 : min(h - h0, WAVE), per = WAVE / heads, mine = lane / heads;
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
                b[u] = e < n_edges ? (int64_t)buckets[e] - b0 : -1;
                x[u] = e < n_edges ? (A)Elem<D>::ld(ds + (PAIRS ? h0 * n_edges + e : e * h + h0 + lane % heads)) : A(0);
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
    const int64_t n = (n_edges + spare) * h;
    hipLaunchKernelGGL((k_bucket_rows<T, O>), dim3((unsigned)((n + BLOCK - 1) / BLOCK)), dim3(BLOCK), 0, s, (const T *)table, buckets, (O *)bias, n_edges, n_buckets, h,
                       (typename Elem<T>::acc_t)factor, spare);
    return launch_status();
}
template <typename D, typename T, typename B>
int run_sums(const void *ds, const B *buckets, void *dtable, void *ws, int64_t n_edges, int64_t n_buckets, int h, double factor, hipStream_t s) {
    using A = typename Elem<D>::acc_t;
    const int parts = sums_parts(n_edges, h);
    const unsigned chunks = sizeof(B) == 2 ? (unsigned)h : (unsigned)((h + WAVE - 1) / WAVE);
    constexpr int WIDE = SUMS_WIDE * 4 / (int)sizeof(A), LONG = SUMS_LONG * 4 / (int)sizeof(A);
    if (n_buckets <= WIDE)
        hipLaunchKernelGGL((k_bucket_sums<D, A, B, 4, WIDE>), dim3(parts, chunks, 1), dim3(4 * WAVE), 4 * WIDE * WAVE * sizeof(A), s, (const D *)ds, buckets, (A *)ws, n_edges,
                           n_buckets, h);
    else
        hipLaunchKernelGGL((k_bucket_sums<D, A, B, 1, LONG>), dim3(parts, chunks, (unsigned)((n_buckets + LONG - 1) / LONG)), dim3(WAVE), LONG * WAVE * sizeof(A), s,
                           (const D *)ds, buckets, (A *)ws, n_edges, n_buckets, h);
    const int st = launch_status();
    if (st != BPT_OK) return st;
    hipLaunchKernelGGL((k_bucket_finish<T, A>), dim3((unsigned)((n_buckets * h + 15) / 16)), dim3(BLOCK), 0, s, (const A *)ws, parts, (T *)dtable, n_buckets * h, (A)factor);
    return launch_status();
}

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
    if (dtype == BPT_F64) return run_sums<double, double, int64_t>(ds, buckets, dtable, workspace, n_edges, n_buckets, h, factor, s);
    if (dtype == BPT_F32) return run_sums<float, float, int64_t>(ds, buckets, dtable, workspace, n_edges, n_buckets, h, factor, s);
    if (ds_dtype == BPT_F32) return run_sums<float, bf16_t, int64_t>(ds, buckets, dtable, workspace, n_edges, n_buckets, h, factor, s);
    return run_sums<bf16_t, bf16_t, int64_t>(ds, buckets, dtable, workspace, n_edges, n_buckets, h, factor, s);
}

int bpt_bucket_pairs_forward(const void *table, const int64_t *buckets, const int32_t *eid_of_pair, uint16_t *codes, float *bias, int64_t n_edges, int64_t n_buckets,
                             int h, double factor, int dtype, void *stream) {
    if (dtype != BPT_F32 && dtype != BPT_BF16) return BPT_ERR_DTYPE;
    if (!is_size(n_edges, n_buckets, h) || n_buckets > NO_BUCKET) return BPT_ERR_SIZE;
    if (n_edges == 0) return BPT_OK;
    if (!table || !buckets || !eid_of_pair || !codes || !bias) return BPT_ERR_NULL;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)((n_edges + BLOCK - 1) / BLOCK));
    hipLaunchKernelGGL(k_bucket_codes, grid, dim3(BLOCK), 0, s, buckets, eid_of_pair, codes, n_edges, n_buckets);
    if (dtype == BPT_F32) hipLaunchKernelGGL((k_bucket_terms<float>), grid, dim3(BLOCK), 0, s, (const float *)table, codes, bias, n_edges, h, (float)factor);
    else hipLaunchKernelGGL((k_bucket_terms<bf16_t>), grid, dim3(BLOCK), 0, s, (const bf16_t *)table, codes, bias, n_edges, h, (float)factor);
    return launch_status();
}

int bpt_bucket_pairs_backward(const float *ds, const uint16_t *codes, void *dtable, void *workspace, int64_t workspace_bytes, int64_t n_edges, int64_t n_buckets, int h,
                              double factor, int dtype, void *stream) {
    if (dtype != BPT_F32 && dtype != BPT_BF16) return BPT_ERR_DTYPE;
    if (!is_size(n_edges, n_buckets, h) || n_buckets > NO_BUCKET) return BPT_ERR_SIZE;
    if (!dtable || (n_edges > 0 && (!ds || !codes))) return BPT_ERR_NULL;
    if (!workspace || workspace_bytes < bpt_bucket_bias_backward_workspace_bytes(n_edges, n_buckets, h, dtype) || !aligned16(workspace)) return BPT_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == BPT_F32) return run_sums<float, float, uint16_t>(ds, codes, dtable, workspace, n_edges, n_buckets, h, factor, s);
    return run_sums<float, bf16_t, uint16_t>(ds, codes, dtable, workspace, n_edges, n_buckets, h, factor, s);
}

}  // extern "C"
