// What libbptattn and libbptscore share: element types, work distribution, the tile kernels of the fused attention (templates,
// instantiated by the launchers of either library), what merges split rows, and the host-side checks of plans and arguments.
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <utility>
#include <vector>

#include "../../include/bptattn.h"

namespace {

constexpr int WAVE = 64;
constexpr int WAVES_PER_BLOCK = 4;
constexpr int BLOCK = WAVE * WAVES_PER_BLOCK;
constexpr float M_INIT_LOG2 = -1.4426950408889634e9f;   // -1e9 (graphop_kernel.cu:428) in base-2 units
constexpr float LOG2E = 1.4426950408889634f;
// Where a running maximum starts.  MOD (score options): a slope times a distance has no bound that scores of products have, and a row whose scores all lie below the
// start would count as empty.
template <bool MOD> constexpr float m_init() { return MOD ? -3.0e38f : M_INIT_LOG2; }

// ------------------------------------------------------------------------------------------
// element types
// ------------------------------------------------------------------------------------------
struct bf16_t { uint16_t bits; };
typedef float floatx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float bf16_to_f32(uint16_t b) { return __uint_as_float(((uint32_t)b) << 16); }
__device__ __forceinline__ uint16_t f32_to_bf16(float f) {
    uint32_t u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);   // NaN stays NaN
    u += 0x7fffu + ((u >> 16) & 1u);                                              // round to nearest even
    return (uint16_t)(u >> 16);
}

template <typename T> struct Elem;
template <> struct Elem<float> {
    using acc_t = float;
    static __device__ __forceinline__ float ld(const float *p) { return *p; }
    static __device__ __forceinline__ void st(float *p, float v) { *p = v; }
};
template <> struct Elem<double> {
    using acc_t = double;
    static __device__ __forceinline__ double ld(const double *p) { return *p; }
    static __device__ __forceinline__ void st(double *p, double v) { *p = v; }
};
template <> struct Elem<bf16_t> {
    using acc_t = float;
    static __device__ __forceinline__ float ld(const bf16_t *p) { return bf16_to_f32(p->bits); }
    static __device__ __forceinline__ void st(bf16_t *p, float v) { p->bits = f32_to_bf16(v); }
};

__device__ __forceinline__ float exp_acc(float x) { return expf(x); }
__device__ __forceinline__ double exp_acc(double x) { return exp(x); }

// ------------------------------------------------------------------------------------------
// work distribution
// ------------------------------------------------------------------------------------------
struct Item { int row, begin, end, slot; };

// Blocks go round-robin to the 8 XCDs; remap so XCD x gets a contiguous run of block indices (of those behind the first `skip`,
// a multiple of 8).
__device__ __forceinline__ int xcd_contiguous_block(int skip = 0) {
    const int nb = gridDim.x - skip, b = blockIdx.x - skip;
    const int q = nb >> 3, rem = nb & 7, x = b & 7, k = b >> 3;
    return x * q + (x < rem ? x : rem) + k;
}

__device__ __forceinline__ bool fetch_item(const bpt_plan &P, Item &it, int waves_per_block = WAVES_PER_BLOCK, int skip = 0) {
    const int w = xcd_contiguous_block(skip) * waves_per_block + (int)(threadIdx.x >> 6);
    if (w >= (int)P.n_items) return false;
    const int4 v = reinterpret_cast<const int4 *>(P.items)[w];
    // the item is the same for all lanes of the wavefront: keep it in scalar registers
    it.row = __builtin_amdgcn_readfirstlane(v.x);
    it.begin = __builtin_amdgcn_readfirstlane(v.y);
    it.end = __builtin_amdgcn_readfirstlane(v.z);
    it.slot = __builtin_amdgcn_readfirstlane(v.w);
    return true;
}

template <typename A> __device__ __forceinline__ A wave_sum(A x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
template <typename A> __device__ __forceinline__ A wave_max(A x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        A y = __shfl_xor(x, o);
        x = x > y ? x : y;
    }
    return x;
}

// Reduction over NW wavefronts of a block (NW == 1: a single wavefront, no LDS, no barrier).
template <typename A, int NW, bool IS_MAX> __device__ __forceinline__ A group_reduce(A x, A *smem) {
    x = IS_MAX ? wave_max(x) : wave_sum(x);
    if (NW == 1) return x;
    const int w = threadIdx.x >> 6;
    __syncthreads();                       // smem may still be read from the previous reduction
    if ((threadIdx.x & 63) == 0) smem[w] = x;
    __syncthreads();
    A r = smem[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) r = IS_MAX ? (r > smem[i] ? r : smem[i]) : r + smem[i];
    return r;
}

// Heads of fewer than 64 columns (6 x 50, 8 x 40), read and written as they are in memory by the NARROW forms of the tile kernels.
// The products keep their 64 columns: quad j of a head (the four columns a lane group position stands for) starts at column
// 4 j, or at d - 4 where that would run over the end of the head.  What a shifted quad repeats of its neighbour, and the quads past
// the end, are zero in both operands of the products over the columns (the members': tile_load16, tile_load_row_bf16; the
// entries': tile_rows_to_operand): a masking -inf in one of the last columns counts once, as in a zero-padded head, where
// zero in one operand alone would make it NaN.  Results are stored from the quads that start inside the head, a repeated column
// twice with one value.  No other head's memory is touched, so what stands there does not matter.
// Against copies padded to 64 columns and 4, 8 or 16 heads (three pads, the output and its gradient, three slices, and the
// padding heads computed with the rest): 33 765 nodes / 576 k edges at 6 x 50 with dropout, forward and backward,
// 508 -> 253 us, of which 38 are copies of q, k, v and o for the backward (Keep); of the 508 copies were 223, the rest two
// padding heads of eight.
struct Narrow {
    int d, heads;              // columns of a head, heads
    int h;                     // heads the layer is padded to where that shows: dropout keys, lse and workspace rows
    int slices;                // workgroups per group
};

// Copies that a NARROW forward writes beside its result, for a backward whose caller may have written to the rows in the meantime:
// q, k and v by workgroups of the forward's own launch that do nothing else, spread evenly between those of the tiles, and the
// result where it is stored.  The forward waits for its gathers and products and leaves much of the memory's rate unused.  Training
// pass at 33 765 nodes, 6 x 50 float32 with dropout: 265.1 us with four copies of their own behind the forward (62 us of them),
// 252.7 so, 215 with none; the copying workgroups first or last, or with loads past the L2, 253.8 to 256.5; stored the ordinary way,
// into the L2 that the tiles' rows want, 265.
struct Keep {
    const char *src[3];
    char *dst[3];              // on 16 bytes; null: no copy of this one (bytes = 0)
    int64_t bytes[3];
    int per_xcd;               // copying workgroups per XCD
    void *o;                   // second copy of the result, or null
};
constexpr int KEEP_CHUNK = 16384;          // bytes a workgroup copies

typedef float floatx4k __attribute__((ext_vector_type(4), aligned(4)));
typedef float floatx4n __attribute__((ext_vector_type(4)));
// What workgroup blockIdx.x of a launch with copying workgroups among it is to do: the number of its tile workgroup, or -1 after it
// has copied its chunk.
template <int THREADS> __device__ __forceinline__ int keep_or_tile(const Keep &keep) {
    if (keep.per_xcd == 0) return (int)blockIdx.x;
    const uint32_t x = blockIdx.x & 7, w = blockIdx.x >> 3, all = gridDim.x >> 3, c = (uint32_t)keep.per_xcd;
    const uint32_t before = (uint32_t)((uint64_t)w * c / all), upto = (uint32_t)((uint64_t)(w + 1) * c / all);
    if (before == upto) return (int)((w - before) * 8 + x);
    // (chosen by conditions, not by an index: indexed, the arguments would be copied to scratch memory by every wavefront)
    int64_t at = (int64_t)(before * 8 + x) * KEEP_CHUNK, left = keep.bytes[0];
    const char *src = keep.src[0];
    char *dst = keep.dst[0];
#pragma unroll
    for (int i = 1; i < 3; ++i) {
        const int64_t past = at - (left + KEEP_CHUNK - 1) / KEEP_CHUNK * KEEP_CHUNK;
        if (past >= 0) { at = past; left = keep.bytes[i]; src = keep.src[i]; dst = keep.dst[i]; }
        else break;
    }
    src += at;
    dst += at;
    left -= at;
    constexpr int U = 4;                                          // loads in flight
    const floatx4k *from = reinterpret_cast<const floatx4k *>(src) + threadIdx.x;
    floatx4n *to = reinterpret_cast<floatx4n *>(dst) + threadIdx.x;
    const int n = (int)min((int64_t)KEEP_CHUNK, max(left, (int64_t)0)) / 16;       // whole 16-byte pieces
    if (n == KEEP_CHUNK / 16) {
#pragma unroll 1
        for (int i = 0; i < KEEP_CHUNK / 16; i += U * THREADS) {
            floatx4k v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = from[i + u * THREADS];
#pragma unroll
            for (int u = 0; u < U; ++u) __builtin_nontemporal_store(floatx4n{v[u][0], v[u][1], v[u][2], v[u][3]}, to + (i + u * THREADS));
        }
        return -1;
    }
    // the last chunk of a tensor, and what is left of no whole number of 16 bytes (up to seven bfloat16)
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const floatx4k v = reinterpret_cast<const floatx4k *>(src)[i];
        reinterpret_cast<floatx4n *>(dst)[i] = floatx4n{v[0], v[1], v[2], v[3]};
    }
    const int64_t end = 16 * (int64_t)n + 2 * (int)threadIdx.x;
    if (end + 2 <= left) *reinterpret_cast<uint16_t *>(dst + end) = *reinterpret_cast<const uint16_t *>(src + end);
    return -1;
}
constexpr int NARROW_HW = 2;   // heads per workgroup (6 x 50: three workgroups of two, none of them half empty)
__device__ __forceinline__ int narrow_col(const Narrow &nw, int quad) { return min(4 * quad, nw.d - 4); }
// whether column e of the quad as loaded is one that the quad before has (or, past the end of the head, any): 4 quad > d - 4 + e
template <bool NARROW> __device__ __forceinline__ bool narrow_again(const Narrow &nw, int quad, int e) {
    return NARROW && quad > (nw.d - 4 + e) >> 2;
}
typedef float floatx4u __attribute__((ext_vector_type(4), aligned(4)));           // such rows start anywhere on 4 bytes
typedef uint32_t uintx2u __attribute__((ext_vector_type(2), aligned(4)));

// The three sums of the fused backward in one launch, four columns per lane (C a multiple of 256, float partials): grid
// (n_a + n_b, C / 256, 2); blocks x < n_a combine rows of list A into YA (z = 0 only), the others rows of list B into YB0
// (z = 0) and YB1 (z = 1).  Every column is added in the order combine_sum_block uses (wave w takes slots w, w + 4, ...;
// the four wave sums in wave order).
template <typename T> __device__ __forceinline__ void store4(T *p, float4 v);
template <> __device__ __forceinline__ void store4<float>(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
template <> __device__ __forceinline__ void store4<bf16_t>(bf16_t *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2((uint32_t)f32_to_bf16(v.x) | ((uint32_t)f32_to_bf16(v.y) << 16),
                                               (uint32_t)f32_to_bf16(v.z) | ((uint32_t)f32_to_bf16(v.w) << 16));
}
template <typename T> __device__ __forceinline__ float4 load4(const T *p);
template <> __device__ __forceinline__ float4 load4<float>(const float *p) { return *reinterpret_cast<const float4 *>(p); }
template <> __device__ __forceinline__ float4 load4<bf16_t>(const bf16_t *p) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u));
}
// The last one to seven slots of a wavefront (those from k on, in steps of WAVES_PER_BLOCK), all asked for before the first is used: a
// launch that adds up the segments of split rows lasts as long as its longest chain of loads, and one after the other these
// are seven round trips of a chain of eight.  f(place, which of them), in order.  Sixteen before them, where there are as many.  L = 8192, k = 4:
// float32 sums 6.3 -> 5.3 us, bfloat16 6.0 -> 4.7; 16 heads at L = 32768, k = 8 28.7 -> 26.8 and the forward (256 segments in its longest row) 14.4 -> 12.6.
__device__ __forceinline__ int combine_left(int k, int ns) { return k < ns ? (ns - k + WAVES_PER_BLOCK - 1) / WAVES_PER_BLOCK : 0; }
template <typename F> __device__ __forceinline__ void combine_tail(int left, F &&f) {
    if (left & 4) { f(0, 0); f(1, 1); f(2, 2); f(3, 3); }
    if (left & 2) { f(4, left & 4); f(5, (left & 4) + 1); }
    if (left & 1) f(6, left & 6);
}
template <typename T, bool NARROW = false>
__device__ __forceinline__ void combine_sum_block4(const int32_t *__restrict__ hv, const float *__restrict__ ws, T *__restrict__ Y, int C,
                                                   bool accumulate = false, int strip = -1, const Narrow &nw = Narrow{}) {
    __shared__ float4 part[WAVES_PER_BLOCK][WAVE];
    const int row = hv[0], s0 = hv[1], ns = hv[2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = ((strip < 0 ? (int)blockIdx.y : strip) * WAVE + lane) * 4;     // strip of 256 columns: the grid's y unless given
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    const float *col = ws + (size_t)s0 * C + j;
    int k = w;
    for (; k + 15 * WAVES_PER_BLOCK < ns; k += 16 * WAVES_PER_BLOCK) {
        float4 t[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) t[u] = *reinterpret_cast<const float4 *>(col + (size_t)(k + u * WAVES_PER_BLOCK) * C);
#pragma unroll
        for (int u = 0; u < 16; ++u) { s.x += t[u].x; s.y += t[u].y; s.z += t[u].z; s.w += t[u].w; }
    }
    if (k + 7 * WAVES_PER_BLOCK < ns) {
        float4 t[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) t[u] = *reinterpret_cast<const float4 *>(col + (size_t)(k + u * WAVES_PER_BLOCK) * C);
#pragma unroll
        for (int u = 0; u < 8; ++u) { s.x += t[u].x; s.y += t[u].y; s.z += t[u].z; s.w += t[u].w; }
        k += 8 * WAVES_PER_BLOCK;
    }
    const int left = combine_left(k, ns);
    float4 t[7];
    combine_tail(left, [&](int u, int nth) { t[u] = *reinterpret_cast<const float4 *>(col + (size_t)(k + nth * WAVES_PER_BLOCK) * C); });
    combine_tail(left, [&](int u, int) { s.x += t[u].x; s.y += t[u].y; s.z += t[u].z; s.w += t[u].w; });
    part[w][lane] = s;
    __syncthreads();
    if (w == 0) {
        float4 r = part[0][lane];
#pragma unroll
        for (int i = 1; i < WAVES_PER_BLOCK; ++i) { r.x += part[i][lane].x; r.y += part[i][lane].y; r.z += part[i][lane].z; r.w += part[i][lane].w; }
        if constexpr (NARROW) {                                   // 64 columns of the partials per head, d of the result
            const int head = j >> 6, col = j & 63;
            T *const at = Y + (size_t)row * (nw.heads * nw.d) + head * nw.d + col;
            const float x[4] = {r.x, r.y, r.z, r.w};
            for (int e = 0; e < 4; ++e)
                if (head < nw.heads && col + e < nw.d) Elem<T>::st(at + e, x[e]);
            return;
        }
        if (accumulate) {
            const float4 y = load4<T>(Y + (size_t)row * C + j);
            r.x += y.x; r.y += y.y; r.z += y.z; r.w += y.w;
        }
        store4<T>(Y + (size_t)row * C + j, r);
    }
}
template <typename T, bool NARROW = false>
__global__ __launch_bounds__(BLOCK) void k_combine_sum3(const int32_t *__restrict__ heavy_a, int n_a, const float *__restrict__ ws_a,
                                                           T *__restrict__ YA, const int32_t *__restrict__ heavy_b,
                                                           const float *__restrict__ ws_b, T *__restrict__ YB0, T *__restrict__ YB1, int C,
                                                           size_t ws_stride_b, Narrow nw) {
    if ((int)blockIdx.x < n_a) {
        if (blockIdx.z == 0) combine_sum_block4<T, NARROW>(heavy_a + 3 * blockIdx.x, ws_a, YA, C, false, -1, nw);
    } else {
        combine_sum_block4<T, NARROW>(heavy_b + 3 * (blockIdx.x - n_a), ws_b + (size_t)blockIdx.z * ws_stride_b, blockIdx.z == 0 ? YB0 : YB1, C,
                                      false, -1, nw);
    }
}

template <int CTRL> __device__ __forceinline__ float dpp_mov(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}

template <int I> __device__ __forceinline__ float quad_lane(float x) { return dpp_mov<I * 0x55>(x); }   // value of lane I of the quad
__device__ __forceinline__ float quad_bcast(float x, int i) {      // the same for an index that is constant after unrolling
    switch (i & 3) {
    case 0: return quad_lane<0>(x);
    case 1: return quad_lane<1>(x);
    case 2: return quad_lane<2>(x);
    default: return quad_lane<3>(x);
    }
}

// Sum over the LPH lanes that hold one head; the result is in all of them.
template <int LPH> __device__ __forceinline__ float head_sum(float x) {
    if constexpr (LPH >= 2) x += dpp_mov<0xB1>(x);    // quad_perm [1,0,3,2]
    if constexpr (LPH >= 4) x += dpp_mov<0x4E>(x);    // quad_perm [2,3,0,1]
    if constexpr (LPH >= 8) x += dpp_mov<0x141>(x);   // row_half_mirror
    if constexpr (LPH >= 16) x += dpp_mov<0x140>(x);  // row_mirror
    if constexpr (LPH >= 32) x += __shfl_xor(x, 16);
    if constexpr (LPH >= 64) x += __shfl_xor(x, 32);
    return x;
}

// The gathers are latency bound: all row loads of a batch must be in flight before the first
// one is consumed.  Without this fence the instruction scheduler interleaves loads and FMAs to
// save registers and waits for every load separately.
__device__ __forceinline__ void issue_loads_first() { __builtin_amdgcn_sched_barrier(0); }

// ---- a node row over the lanes of a wavefront (the kernels that walk single rows) ----
template <typename T, int H_, int D_> struct Lay {
    static constexpr int H = H_, D = D_, C = H_ * D_;
    static constexpr int LPH = 64 / H_;                 // lanes per head
    static constexpr int EPL = C / 64;                  // elements per lane (all of one head)
    static constexpr int VE = 16 / (int)sizeof(T);      // elements per 16-byte vector
    static constexpr int NV = EPL / VE;                 // 16-byte vectors per lane
    static_assert(64 % H_ == 0 && C % 64 == 0 && EPL % VE == 0 && NV >= 1, "unsupported fast shape");
    static_assert(LPH >= 4, "the row-group kernels broadcast per-member values inside quads of one head");
    static_assert(D_ == NV * LPH * VE, "layout does not tile the head");
    // element offset inside a node row of vector i of `lane`: LPH consecutive lanes cover
    // LPH*16 contiguous bytes of their head
    static __device__ __forceinline__ int off(int lane, int i) { return (lane / LPH) * D + (i * LPH + lane % LPH) * VE; }
};

template <typename T, int H, int D>
__device__ __forceinline__ void load_row(const T *__restrict__ row, int lane, float (&out)[Lay<T, H, D>::EPL]) {
    using L = Lay<T, H, D>;
#pragma unroll
    for (int i = 0; i < L::NV; ++i) {
        if constexpr (sizeof(T) == 4) {
            const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(row) + L::off(lane, i));
            out[4 * i] = v.x; out[4 * i + 1] = v.y; out[4 * i + 2] = v.z; out[4 * i + 3] = v.w;
        } else {
            const uint4 v = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(row) + L::off(lane, i));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                out[8 * i + 2 * c] = __uint_as_float(w[c] << 16);
                out[8 * i + 2 * c + 1] = __uint_as_float(w[c] & 0xffff0000u);
            }
        }
    }
}

template <typename T, int H, int D>
__device__ __forceinline__ void store_row(T *__restrict__ row, int lane, const float (&in)[Lay<T, H, D>::EPL]) {
    using L = Lay<T, H, D>;
#pragma unroll
    for (int i = 0; i < L::NV; ++i) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(reinterpret_cast<float *>(row) + L::off(lane, i)) =
                make_float4(in[4 * i], in[4 * i + 1], in[4 * i + 2], in[4 * i + 3]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                w[c] = (uint32_t)f32_to_bf16(in[8 * i + 2 * c]) | ((uint32_t)f32_to_bf16(in[8 * i + 2 * c + 1]) << 16);
            *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(row) + L::off(lane, i)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// f32 partial rows in the workspace are stored in natural column order (the combine kernels
// index them by column), whatever the element type of the node tensors
template <typename T, int H, int D>
__device__ __forceinline__ void store_row_ws(float *__restrict__ row, int lane, const float (&in)[Lay<T, H, D>::EPL]) {
    using L = Lay<T, H, D>;
#pragma unroll
    for (int i = 0; i < L::NV; ++i)
#pragma unroll
        for (int c = 0; c < L::VE / 4; ++c)
            *reinterpret_cast<float4 *>(row + L::off(lane, i) + 4 * c) =
                make_float4(in[L::VE * i + 4 * c], in[L::VE * i + 4 * c + 1], in[L::VE * i + 4 * c + 2], in[L::VE * i + 4 * c + 3]);
}

template <int N> __device__ __forceinline__ float dot_n(const float (&a)[N], const float (&b)[N]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(a[i], b[i], s);
    return s;
}

// NW wavefronts (a workgroup) share an item: each takes whole batches of its edges, as many as the others, and the sums meet in
// LDS.  False: no such item (the whole workgroup).  parts: how many wavefronts have edges (one at least).
template <int NW, int BATCH> __device__ __forceinline__ bool fetch_item_part(const bpt_plan &P, Item &it, int &part, int &parts) {
    part = 0;
    parts = 1;
    if constexpr (NW == 1) return fetch_item(P, it);
    const int w = xcd_contiguous_block();
    if (w >= (int)P.n_items) return false;
    const int4 v = reinterpret_cast<const int4 *>(P.items)[w];
    it.row = __builtin_amdgcn_readfirstlane(v.x);
    it.begin = __builtin_amdgcn_readfirstlane(v.y);
    it.end = __builtin_amdgcn_readfirstlane(v.z);
    it.slot = __builtin_amdgcn_readfirstlane(v.w);
    const int deg = it.end - it.begin, per = (deg + NW * BATCH - 1) / (NW * BATCH) * BATCH;
    part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    parts = max(1, (deg + max(per, 1) - 1) / max(per, 1));
    it.begin = min(it.begin + part * per, it.end);
    it.end = min(it.begin + per, it.end);
    return true;
}

// Whether a row's softmax has a denominator.  MOD (ScoreMod, below): NaN is one, the row is NaN then.
template <bool MOD> __device__ __forceinline__ bool has_sum(float l) { return MOD ? l != 0.f : l > 0.f; }

// Combine the (m, l, acc) partials of each split row.  Grid (n_heavy, C / 64): one block per split row
// and 64-column strip; wave w folds slots w, w+4, ... with a running maximum (one pass, eight
// independent loads per step), then the four wave results are merged in wave order.
template <typename T, int HC, int D, bool NARROW = false, bool MOD = false>
__global__ __launch_bounds__(BLOCK) void k_attn_fwd_combine(const int32_t *__restrict__ heavy, const float *__restrict__ ws_acc,
                                                            const float *__restrict__ ws_ml, T *__restrict__ o, float *__restrict__ lse,
                                                            Narrow nw, T *__restrict__ o_keep = nullptr) {
    static_assert(HC * D % WAVE == 0, "strip width");
    const int H = NARROW ? nw.h : HC, C = H * D;                 // (NARROW: one strip per real head)
    __shared__ float pm[WAVES_PER_BLOCK][WAVE], pl[WAVES_PER_BLOCK][WAVE], pa[WAVES_PER_BLOCK][WAVE];
    const int row = heavy[3 * blockIdx.x], s0 = heavy[3 * blockIdx.x + 1], ns = heavy[3 * blockIdx.x + 2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int j = blockIdx.y * WAVE + lane, head = j / D;
    const float *ml = ws_ml + ((size_t)s0 * H + head) * 2;      // slot stride 2*H
    const float *col = ws_acc + (size_t)s0 * C + j;              // slot stride C
    float M = m_init<MOD>(), lsum = 0.f, a = 0.f;
    int kk = w;
    float tm[16], tl[16], ta[16];
    auto ask = [&](int u, int nth) {
        const size_t sl = (size_t)(kk + nth * WAVES_PER_BLOCK);
        tm[u] = ml[sl * 2 * H];
        tl[u] = ml[sl * 2 * H + 1];
        ta[u] = col[sl * C];
    };
    auto fold = [&](auto n) {
        float mx = M;
#pragma unroll
        for (int u = 0; u < n(); ++u) mx = fmaxf(mx, tm[u]);
        const float resc = __builtin_amdgcn_exp2f(M - mx);
        lsum *= resc;
        a *= resc;
#pragma unroll
        for (int u = 0; u < n(); ++u) {
            const float wgt = __builtin_amdgcn_exp2f(tm[u] - mx);
            lsum = fmaf(tl[u], wgt, lsum);
            a = fmaf(ta[u], wgt, a);
        }
        M = mx;
    };
    for (; kk + 15 * WAVES_PER_BLOCK < ns; kk += 16 * WAVES_PER_BLOCK) {
#pragma unroll
        for (int u = 0; u < 16; ++u) ask(u, u);
        fold(std::integral_constant<int, 16>{});
    }
    if (kk + 7 * WAVES_PER_BLOCK < ns) {
#pragma unroll
        for (int u = 0; u < 8; ++u) ask(u, u);
        fold(std::integral_constant<int, 8>{});
        kk += 8 * WAVES_PER_BLOCK;
    }
    const int left = combine_left(kk, ns);
    if (left > 0) {
#pragma unroll
        for (int u = 0; u < 7; ++u) { tm[u] = -INFINITY; tl[u] = ta[u] = 0.f; }
        combine_tail(left, ask);
        fold(std::integral_constant<int, 7>{});
    }
    pm[w][lane] = M; pl[w][lane] = lsum; pa[w][lane] = a;
    __syncthreads();
    if (w == 0) {
        float Mx = pm[0][lane];
#pragma unroll
        for (int i = 1; i < WAVES_PER_BLOCK; ++i) Mx = fmaxf(Mx, pm[i][lane]);
        float L = 0.f, A = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES_PER_BLOCK; ++i) {
            const float wgt = __builtin_amdgcn_exp2f(pm[i][lane] - Mx);
            L = fmaf(pl[i][lane], wgt, L);
            A = fmaf(pa[i][lane], wgt, A);
        }
        if (!NARROW) Elem<T>::st(o + (size_t)row * C + j, has_sum<MOD>(L) ? A / L : 0.f);
        else if (lane < nw.d) {
            Elem<T>::st(o + (size_t)row * (nw.heads * nw.d) + head * nw.d + lane, has_sum<MOD>(L) ? A / L : 0.f);
            if (o_keep) Elem<T>::st(o_keep + (size_t)row * (nw.heads * nw.d) + head * nw.d + lane, has_sum<MOD>(L) ? A / L : 0.f);
        }
        if (j % D == 0) lse[(size_t)row * H + head] = has_sum<MOD>(L) ? Mx + log2f(L) : 0.f;
    }
}

// Dropout on the attention probabilities (modules/attention.py:73): the keep / drop decision of (pair n, head h) is
// a hash of n * H + h and the call's seed, so that forward and backward agree without storing a mask.  n is the
// pair's number in the destination-side groups (entry's first pair + rank of the member in the entry's mask).
// Returns the multiplier 1 / (1 - p) or 0.
__device__ __forceinline__ float dropout_keep(uint32_t key, uint32_t seed, uint32_t thr, float inv_keep) {
    uint32_t x = key ^ seed;
    x ^= x >> 16; x *= 0x7feb352du; x ^= x >> 15; x *= 0x846ca68bu; x ^= x >> 16;
    return x >= thr ? inv_keep : 0.f;
}

// by how much (base-2 units) a score may exceed the exponent reference of its row before the reference is raised (row groups and tiles)
constexpr float MFMA_TAU = 8.f;

__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

typedef short bf16x4_t __attribute__((ext_vector_type(4)));
// two registers of bfloat16 pairs as the four-element operand of the bfloat16 matrix instructions
__device__ __forceinline__ bf16x4_t as_bf16x4(uint32_t a, uint32_t b) {
    const uint2 u = make_uint2(a, b);
    return __builtin_bit_cast(bf16x4_t, u);
}

// ---- dense tiles: groups of 16 rows, one wavefront per head ---------------------------------------------------------
// A group of TILE_R = 16 rows (or row segments) and its entries (the union of the members' neighbours, each with a
// 16-bit member mask) is walked in blocks of 16 entries as a dense 16 x 16 problem on the matrix cores: the pairs a
// block does not have are computed and masked.  Adjacent rows of a BPT graph share most neighbours (35 % of a block's
// pairs exist at L = 8192, k = 4), and a dense block costs 4 cycles per pair and head in float32 against 25-35 issue
// slots of the gather form.  Workgroup = H wavefronts, wavefront = one head, so every lane keeps 1/64 of a
// 16 x 64 tile per operand and nothing is exchanged between wavefronts.
//
// v_mfma_f32_16x16x4f32: D[i][n] += sum_k A[i][k] B[k][n], lane (c = lane % 16, g = lane / 16) supplies A[c][g] and
// B[g][c] and holds D[4 g + r][c] in register r.  Which column of a row a (step, g) pair stands for is free as long as
// A and B agree, so operands are held as 16-byte vectors (the members' rows are loaded that way; the entries' rows
// reach the first layout below through LDS, see tile_rows_to_operand):
//   scores S^T = K Q^T : A = K[entry e(c)][16 t + 4 g + e], B = q[member c][16 t + 4 g + e] (steps t, e = 0..3), where
//                        row c of the product is entry e(c) = 4 (c % 4) + c / 4 of the block, so that
//                        register r of lane (c, g) = score of (entry 4 r + g, member c);
//   output O += P V    : A = register r of the probabilities as they stand (row = member c, k = g stands for entry
//                        4 r + g), B = V[entry 4 r + g][4 c + nb]; register r' of accumulator nb of lane (c, g) =
//                        O[member 4 g + r'][4 c + nb]: four consecutive columns per lane, 256 contiguous bytes per
//                        member and 16 lanes.  Step r of such a product covers the neighbouring entries 4 r .. 4 r + 3:
//                        past the end of a group's entry list (half of its last block on average) steps are left out.
//   (The bfloat16 kernels below keep entry 4 g + r in register r: their products over the entries are one instruction.)
// Softmax state is per lane for member c (the four lanes of a member hold partial denominators that are added at the
// end); the exponent reference is raised lazily as in the matrix-core forward above.
constexpr int TILE_R = 16;
constexpr int TILE_CHUNK = 128;                     // entries staged in LDS at a time = 8 blocks

typedef float floatx4v __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2v __attribute__((ext_vector_type(2)));

typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef float floatx2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    union { bf16x2v v; uint32_t u; } r;
    r.v = __builtin_convertvector(floatx2v{lo, hi}, bf16x2v);      // round to nearest even
    return r.u;
}

// What a tile costs beside its blocks - sums and maxima over lane groups, the rows it stores, masks - is kept to few vector instructions:
// float32 products (v_mfma_f32_16x16x4) and vector arithmetic do not run side by side on a SIMD, whichever wavefronts they come from (a
// wavefront of each takes the sum of their times: 288 + 351 -> 628 cycles; bfloat16 16 x 16 x 32 products 145 + 345 -> 405).  Lane groups
// are swapped instead of looked up through the LDS crossbar, masks are one bit field extract and one and, a member's row or slot is one
// word, rows go to 32-bit offsets from a uniform base, bfloat16 is rounded by the hardware and sums that are still zero are not rescaled;
// the float32 destination side reads masks and pair numbers back from LDS and no longer spills.  Same results to the bit.  Kernels before ->
// after, forward / destination / source side: bfloat16, L = 8192, k = 4 18.5 / 25.6 / 29.2 -> 17.1 / 24.6 / 26.5 us, 16 heads at L = 32768, k = 8
// 185 / 241 / 339 -> 184 / 240 / 333; float32, L = 8192 35.3 / 59.3 / 42.8 -> 34.1 / 58.1 / 40.9, 32-graph batch 68.6 / 105.1 / 89.4 -> 67.0 / 101.6 / 87.4.
// x of the lanes c, 16 + c, 32 + c and 48 + c, combined, in all four of them
__device__ __forceinline__ float groups_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float groups_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// x where bit `bit` of the mask is set, -inf (0) where it is not
__device__ __forceinline__ float where_pair(int mask, int bit, float x) {
    const int m = __builtin_amdgcn_sbfe(mask, bit, 1);
    return __int_as_float((__float_as_int(x) & m) | (0xff800000 & ~m));
}
__device__ __forceinline__ float where_pair_or_zero(int mask, int bit, float x) {
    return __int_as_float(__float_as_int(x) & __builtin_amdgcn_sbfe(mask, bit, 1));
}
__device__ __forceinline__ float lane_bcast(float x, int src_lane) {
    return __int_as_float(__builtin_amdgcn_ds_bpermute(src_lane << 2, __float_as_int(x)));
}
__device__ __forceinline__ int lane_bcast(int x, int src_lane) { return __builtin_amdgcn_ds_bpermute(src_lane << 2, x); }

// Common start of the tile kernels.  HW heads (= wavefronts) per workgroup: workgroup b handles head slice
// (b / 8) % (H / HW) of group (b / 8) / (H / HW) of XCD b % 8's range.
struct TileCtx {
    int lane, wv, c, g, head, p_begin, p_end, part, grp;
    int2 member;                 // (row, slot) of member c
    uint32_t offa, offv;         // byte offsets of this lane inside a node row: its 16-column slice of the head (operands of the
                                 // products that contract over columns, + 64 t bytes per step), and its columns 4 c .. 4 c + 3
};

template <typename T, int H, int D, int HW, bool NARROW = false, int SP = 1>
__device__ __forceinline__ bool tile_begin(const bpt_plan &P, TileCtx &t, const Narrow &nw, unsigned block = blockIdx.x) {
    static_assert(D == 64 && (H * SP) % HW == 0 && HW % SP == 0 && (sizeof(T) == 4 || sizeof(T) == 2), "64 columns per head: one 16-column slice per lane group");
    static_assert(!NARROW || SP == 1 || SP == HW, "heads a workgroup has past the last one leave its barrier alone");
    constexpr int HEADS = HW / SP;
    const int HS = NARROW ? nw.slices : H / HEADS;
    t.lane = threadIdx.x & (WAVE - 1);
    t.wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    t.c = t.lane & 15;
    t.g = t.lane >> 4;
    const int x = block & 7, w = (int)(block >> 3) / HS;
    const int grp = __builtin_amdgcn_readfirstlane(P.grp_chunks[x]) + w;
    if (grp >= __builtin_amdgcn_readfirstlane(P.grp_chunks[x + 1])) return false;
    t.grp = grp;
    t.member = reinterpret_cast<const int2 *>(P.grp_members)[(size_t)grp * TILE_R + t.c];
    t.p_begin = __builtin_amdgcn_readfirstlane(P.grp_ptr[grp]);
    t.p_end = __builtin_amdgcn_readfirstlane(P.grp_ptr[grp + 1]);
    t.part = SP > 1 ? t.wv / HEADS : 0;
    if constexpr (SP > 1) {
        const int per = ((t.p_end - t.p_begin + TILE_R * SP - 1) / (TILE_R * SP)) * TILE_R;
        t.p_begin = min(t.p_begin + t.part * per, t.p_end);
        t.p_end = min(t.p_begin + per, t.p_end);
    }
    t.head = (int)((block >> 3) % HS) * HEADS + (SP > 1 ? t.wv % HEADS : t.wv);
    if (NARROW) {
        if (t.head >= nw.heads) return false;
        t.offa = (uint32_t)(t.head * nw.d * sizeof(T));
        t.offv = (uint32_t)((t.head * nw.d + narrow_col(nw, t.c)) * sizeof(T));
        return true;
    }
    t.offa = (uint32_t)((t.head * D + 4 * t.g) * sizeof(T));
    t.offv = (uint32_t)((t.head * D + 4 * t.c) * sizeof(T));
    return true;
}

// The entry list of a group is staged, TILE_CHUNK entries at a time, in a wavefront-private piece of LDS as (neighbour,
// mask) pairs: every lane needs five of them per block (its A-operand row and the four rows / masks of its lane
// group), which would otherwise be five dependent global loads in front of every block's row loads.
struct TileEntryRegs {
    int4 x[TILE_CHUNK / WAVE];
};
// first half: the loads.  A kernel asks for its first piece before it reads its members' rows, so that the two round trips
// run side by side; in source order the compiler puts the members' arithmetic (and its wait) in front of these loads.
__device__ __forceinline__ void tile_ask_entries(const bpt_plan &P, int p0, int cnt, int lane, TileEntryRegs &r) {
    const int4 *entries = reinterpret_cast<const int4 *>(P.grp_entries);
#pragma unroll
    for (int u = 0; u < TILE_CHUNK / WAVE; ++u) r.x[u] = entries[p0 + min(u * WAVE + lane, cnt - 1)];   // past the end: the last entry again
}
// second half: into the wavefront's piece of LDS
__device__ __forceinline__ void tile_put_entries(const TileEntryRegs &r, int2 *lds, int cnt, int lane, int *first = nullptr) {
#pragma unroll
    for (int u = 0; u < TILE_CHUNK / WAVE; ++u) {
        const int e = u * WAVE + lane;
        int nbr = r.x[u].x, mask = r.x[u].y;
        asm volatile("" : "+v"(nbr), "+v"(mask));                 // (the values are used from here on: nothing of this half moves up to the loads)
        lds[e] = make_int2(nbr, e < cnt ? mask : 0);              // past the end: an empty mask
        if (first) first[e] = r.x[u].z;                          // number of the entry's first pair (members follow in ascending order)
    }
    wave_lds_fence();
}
__device__ __forceinline__ void tile_stage_entries(const bpt_plan &P, int2 *lds, int p0, int cnt, int lane, int *first = nullptr) {
    TileEntryRegs r;
    tile_ask_entries(P, p0, cnt, lane, r);
    tile_put_entries(r, lds, cnt, lane, first);
}
// number of the pair (entry, member c) among the plan's pairs: the entry's first pair + the members before c in its mask
__device__ __forceinline__ int tile_pair_number(int first, int mask, int c) { return first + __popc((uint32_t)mask & ((1u << c) - 1u)); }

// this lane's 16 columns of a node row (bytes offa + 64 t), as the A or B operand of a product over columns
template <bool NARROW>
__device__ __forceinline__ floatx4v tile_load4(const char *row, int t, int g, const Narrow &nw) {      // the four of step t
    if constexpr (NARROW) {
        const int quad = 4 * (4 * t + g), col = min(quad, nw.d - 4);
        const floatx4u x = *reinterpret_cast<const floatx4u *>(row + 4 * col);
        return floatx4v{col >= quad ? x[0] : 0.f, col + 1 >= quad ? x[1] : 0.f, col + 2 >= quad ? x[2] : 0.f, col + 3 >= quad ? x[3] : 0.f};
    } else {
        return *reinterpret_cast<const floatx4v *>(row + 64 * t);
    }
}
template <bool NARROW>
__device__ __forceinline__ void tile_load16(const char *row, float (&out)[16], int g, const Narrow &nw) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const floatx4v x = tile_load4<NARROW>(row, t, g, nw);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[4 * t + e] = x[e];
    }
}
// this lane's four columns of an entry's row
template <bool NARROW> __device__ __forceinline__ float4 tile_row4(const char *p) {
    if constexpr (NARROW) {
        const floatx4u x = *reinterpret_cast<const floatx4u *>(p);
        return make_float4(x[0], x[1], x[2], x[3]);
    } else {
        return *reinterpret_cast<const float4 *>(p);
    }
}

// register r of the result of lane (c, g) = sum over the 64 columns of a[row 4 g + r] * b[member c], a[row c] = what lane c passes
__device__ __forceinline__ floatx4v tile_dot(const float (&a)[16], const float (&b)[16]) {
    floatx4v s0 = floatx4v{0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
        s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i + 1], b[i + 1], s1, 0, 0, 0);
    }
    return s0 + s1;
}

// acc[nb][r'] (member 4 g + r', column 4 c + nb) += sum over the block's entries of w[member][entry] * row[entry][column]:
// w = this lane's four weights (member c with entries 4 r + g), rows = columns 4 c .. 4 c + 3 of the rows of entries 4 r + g.
// Step r of the product stands for the four NEIGHBOURING entries 4 r .. 4 r + 3 (one per lane group), so a step whose
// entries lie past the end of the group's list (nv = the block's entries that exist) is left out.
__device__ __forceinline__ void tile_axpy_upto(const float (&w)[4], const float4 (&rows)[4], floatx4v (&acc)[4], int nv) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (4 * r < nv) {
            acc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r], rows[r].x, acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r], rows[r].y, acc[1], 0, 0, 0);
            acc[2] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r], rows[r].z, acc[2], 0, 0, 0);
            acc[3] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r], rows[r].w, acc[3], 0, 0, 0);
        } else {
            // (the step's rows are marked as read: left in flight, they would make the next block's loads wait for
            // everything that is outstanding, this block's stores included)
            asm volatile("" ::"v"(rows[r].x), "v"(rows[r].y), "v"(rows[r].z), "v"(rows[r].w));
        }
    }
}

// The members' result rows: whole rows go to `out` (scaled by inv[member] where given), segments of split rows to the
// workspace in natural column order.  Whole rows are written past the L2 (non-temporal): this kernel does not read them again,
// and written the ordinary way they push out the neighbours' rows that the other tiles of the XCD are about to read.  Sum of a
// training step's kernels, new inputs every pass, before -> now: 32-graph batch float32 284 -> 274 us (forward 76 -> 70.5),
// L = 8192 float32 161 -> 157, bfloat16 91 -> 85.5 (forward 21.8 -> 19.2), L = 32768, k = 4 649 -> 632, window 128 97 -> 94.5;
// L = 512 level.  The same on the stores of (p, ds), which the source side reads soon, or on its loads of them: 47 -> 50.5 and
// 47 -> 55 us for the source side of L = 8192; on the loads of the members' rows: destination side 58 -> 61.6.
// where: per member, its row, -1 where there is none, -2 - slot for a segment of a split row (tile_where of lane c for member c)
__device__ __forceinline__ int tile_where(int2 member) { return member.x < 0 ? -1 : member.y < 0 ? member.x : -2 - member.y; }
template <int H, int D, bool SCALE, bool NARROW, typename T>
__device__ __forceinline__ void tile_store_row(const TileCtx &t, int r, float4 x, float inv_c, T *__restrict__ out, float *__restrict__ ws,
                                               const Narrow &nw, int where, T *__restrict__ also = nullptr) {      // also (NARROW): second copy of whole rows
    const int m = 4 * t.g + r;                                    // the member whose row this lane stores a piece of
    int at = lane_bcast(where, m);
    const float inv = SCALE ? lane_bcast(inv_c, m) : 1.f;
    if (NARROW && 4 * t.c >= nw.d) at = -1;
    const int col = NARROW ? narrow_col(nw, t.c) : 4 * t.c;
    if (at >= 0) {
        if (SCALE) { x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv; }
        // (node tensors end before 4 GiB)
        const uint32_t off = NARROW ? ((uint32_t)at * (uint32_t)(nw.heads * nw.d) + (uint32_t)(t.head * nw.d + col)) * (uint32_t)sizeof(T)
                                    : (uint32_t)at * (uint32_t)(H * D * sizeof(T)) + t.offv;
        char *const to = reinterpret_cast<char *>(out) + off;
        if constexpr (sizeof(T) == 4) {
            if constexpr (NARROW) {
                *reinterpret_cast<floatx4u *>(to) = floatx4u{x.x, x.y, x.z, x.w};
                if (also) *reinterpret_cast<floatx4u *>(reinterpret_cast<char *>(also) + off) = floatx4u{x.x, x.y, x.z, x.w};
            } else __builtin_nontemporal_store(floatx4v{x.x, x.y, x.z, x.w}, reinterpret_cast<floatx4v *>(to));
        } else {
            const uint2 y = make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
            if constexpr (NARROW) {
                *reinterpret_cast<uintx2u *>(to) = uintx2u{y.x, y.y};
                if (also) *reinterpret_cast<uintx2u *>(reinterpret_cast<char *>(also) + off) = uintx2u{y.x, y.y};
            } else __builtin_nontemporal_store(uintx2v{y.x, y.y}, reinterpret_cast<uintx2v *>(to));
        }
    } else if (at < -1) {
        float *const to = ws + (size_t)(-2 - at) * (NARROW ? nw.h * D : H * D) + t.head * D + col;
        if constexpr (NARROW) *reinterpret_cast<floatx4u *>(to) = floatx4u{x.x, x.y, x.z, x.w};
        else *reinterpret_cast<float4 *>(to) = x;
    }
}
template <int H, int D, bool SCALE, bool NARROW, typename T>
__device__ __forceinline__ void tile_store_rows(const TileCtx &t, const floatx4v (&acc)[4], float inv_c, T *__restrict__ out,
                                                float *__restrict__ ws, const Narrow &nw, T *__restrict__ also = nullptr) {
    const int where = tile_where(t.member);
#pragma unroll
    for (int r = 0; r < 4; ++r)
        tile_store_row<H, D, SCALE, NARROW>(t, r, make_float4(acc[0][r], acc[1][r], acc[2][r], acc[3][r]), inv_c, out, ws, nw, where, also);
}

// SP > 1: SP wavefronts of a workgroup share a tile and head, each walks a contiguous SP-th of the tile's blocks (tile_begin),
// and what they have summed up meets in LDS: every wavefront leaves its accumulators in its own piece, [r][lane] so that
// the 16-byte accesses of a wavefront are contiguous, and after one barrier adds up and stores the members 4 g + r of its
// 4 / SP registers r.  Parts are added in their order: the same bits on every run.
constexpr int TILE_PART_FLOATS = TILE_R * 64;                     // accumulators of a wavefront
__device__ __forceinline__ void tile_park(float *part, const floatx4v (&acc)[4], int lane) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
        *reinterpret_cast<floatx4v *>(part + (r * WAVE + lane) * 4) = floatx4v{acc[0][r], acc[1][r], acc[2][r], acc[3][r]};
}
// sum over the parts of register r, part s (`stride` floats after part s - 1) weighted with wgt[s] of the lane's member
template <int SP, bool WEIGHTED>
__device__ __forceinline__ float4 tile_meet(const float *part0, int stride, int r, const TileCtx &t, const float (&wgt)[SP]) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int s = 0; s < SP; ++s) {
        const floatx4v y = *reinterpret_cast<const floatx4v *>(part0 + s * stride + (r * WAVE + t.lane) * 4);
        if constexpr (WEIGHTED) {
            const float w = lane_bcast(wgt[s], 4 * t.g + r);
            x.x = fmaf(w, y[0], x.x); x.y = fmaf(w, y[1], x.y); x.z = fmaf(w, y[2], x.z); x.w = fmaf(w, y[3], x.w);
        } else {
            x.x += y[0]; x.y += y[1]; x.z += y[2]; x.w += y[3];
        }
    }
    return x;
}
// the same for a kernel without weights: parked accumulators of the SP parts -> result rows
template <int SP, int H, int D, bool NARROW, typename T>
__device__ __forceinline__ void tile_meet_and_store(const float *part0, int stride, const TileCtx &t, T *__restrict__ out, float *__restrict__ ws,
                                                    const Narrow &nw) {
    constexpr int RS = 4 / SP;
    const float none[SP] = {};
#pragma unroll
    for (int i = 0; i < RS; ++i) {
        const int r = t.part * RS + i;
        tile_store_row<H, D, false, NARROW>(t, r, tile_meet<SP, false>(part0, stride, r, t, none), 1.f, out, ws, nw, tile_where(t.member));
    }
}
// ... and for the forward: with the parts' exponent references and denominators (left behind the accumulators by member)
constexpr int TILE_PART_FWD_FLOATS = TILE_PART_FLOATS + 2 * TILE_R;
template <int SP, int H, int D, bool NARROW, bool MOD, typename T>
__device__ __forceinline__ void tile_meet_forward(float *mine, const float *part0, int stride, const TileCtx &t, const floatx4v (&acc)[4], float &mref,
                                                  float &lt, T *__restrict__ out, float *__restrict__ ws, const Narrow &nw,
                                                  T *__restrict__ also) {
    constexpr int RS = 4 / SP;
    tile_park(mine, acc, t.lane);
    if (t.g == 0) {
        mine[TILE_PART_FLOATS + 2 * t.c] = mref;
        mine[TILE_PART_FLOATS + 2 * t.c + 1] = lt;
    }
    __syncthreads();
    float wgt[SP], l = 0.f, M = m_init<MOD>();
#pragma unroll
    for (int s = 0; s < SP; ++s) {
        wgt[s] = part0[s * stride + TILE_PART_FLOATS + 2 * t.c];
        M = fmaxf(M, wgt[s]);
    }
#pragma unroll
    for (int s = 0; s < SP; ++s) {
        wgt[s] = __builtin_amdgcn_exp2f(wgt[s] - M);
        l = fmaf(wgt[s], part0[s * stride + TILE_PART_FLOATS + 2 * t.c + 1], l);
    }
    mref = M;
    lt = l;
    const float inv = has_sum<MOD>(l) ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < RS; ++i) {
        const int r = t.part * RS + i;
        tile_store_row<H, D, true, NARROW>(t, r, tile_meet<SP, true>(part0, stride, r, t, wgt), inv, out, ws, nw, tile_where(t.member), also);
    }
}

// Edge ids of this lane's four pairs of a block, (entry first_entry + step * r, member c): what the dropout hash and the score term are
// indexed by (n_edges, the spare row, where the pair does not exist; past the group's end the last entry is read again).
__device__ __forceinline__ void tile_pair_eids(const bpt_plan &P, int first_entry, int p_end, int c, int (&xe)[4], int step = 1) {
#pragma unroll
    for (int r = 0; r < 4; ++r) xe[r] = P.grp_eids[(size_t)min(first_entry + step * r, p_end - 1) * TILE_R + c];
}
// Which entry of a block lane c loads as row c of the products over the columns, in the float32 tile kernels: the
// scores of entries 4 r + g have to come out in register r of lane group g (row 4 g + r of the product), so that step r
// of the products over the entries stands for four NEIGHBOURING entries and can be left out past the end of the list.
__device__ __forceinline__ int tile_entry_of_row(int c) { return 4 * (c & 3) + (c >> 2); }
// Where the score term of the pair (entry, member c) sits and its gradient goes.  BIAS == 1, stored by edge id: row eid
// of (n_edges + 1, H), the spare last row for a pair that does not exist.  BIAS == 2, stored in the plan's own order:
// head-major at the pair's number, x[head * n_edges + number]: the lanes of an entry touch one run of memory and no
// index is read on the way; a pair that does not exist gets a neighbour's place, which is read and not used.
template <int H, int BIAS>
__device__ __forceinline__ uint32_t tile_bias_at(const bpt_plan &P, int head, int eid, int number) {
    if constexpr (BIAS == 2) return (uint32_t)head * (uint32_t)P.n_edges + (uint32_t)min(number, (int)P.n_edges - 1);
    else return (uint32_t)eid * (uint32_t)H + (uint32_t)head;
}

// The rows of a block's entries come from memory in the layout of the products over the entries (lane (c, g): columns
// 4 c .. 4 c + 3 of the rows of entries 4 r + g: the sixteen lanes of a lane group read one row's 256 contiguous bytes).
// The products over the COLUMNS want lane c to hold sixteen columns of ONE row (entry tile_entry_of_row(c)); loaded that
// way, neighbouring lanes read different rows and the texture addresser spends four cycles on every group of four lanes
// instead of one.  So the rows are loaded once, in the first layout, and turned in a wavefront-private piece of LDS:
// rows of TILE_KT_STRIDE floats (64 + 4: the sixteen rows of a read fall on different banks).
constexpr int TILE_KT_STRIDE = 68;
template <bool NARROW>
__device__ __forceinline__ void tile_rows_to_operand(float *kt, const float4 (&rows)[4], int c, int g, float (&out)[16], const Narrow &nw) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
        *reinterpret_cast<floatx4v *>(kt + (4 * r + g) * TILE_KT_STRIDE + 4 * c) =
            floatx4v{narrow_again<NARROW>(nw, c, 0) ? 0.f : rows[r].x, narrow_again<NARROW>(nw, c, 1) ? 0.f : rows[r].y,
                     narrow_again<NARROW>(nw, c, 2) ? 0.f : rows[r].z, narrow_again<NARROW>(nw, c, 3) ? 0.f : rows[r].w};
    wave_lds_fence();
    const float *src = kt + tile_entry_of_row(c) * TILE_KT_STRIDE + 4 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const floatx4v x = *reinterpret_cast<const floatx4v *>(src + 16 * t);
        out[4 * t] = x[0]; out[4 * t + 1] = x[1]; out[4 * t + 2] = x[2]; out[4 * t + 3] = x[3];
    }
    wave_lds_fence();                                             // (read before the next block's rows are written)
}

// The members' rows likewise: lane (c, g) asks for columns 4 c .. 4 c + 3 of the row of member 4 g + r, and tile_rows_to_operand gives lane c
// the row of member c: 16 cycles of the texture addresser a load instead of 64.  Destination side, 32-graph batch 102.8 -> 99.7 us, 6 x 50 with
// dropout 90.9 -> 87.4 and its forward 97.9 -> 96.4, L = 8192, k = 4 level.  (The forward that asks for its K rows a block ahead has no
// registers for it: asked for with the entries and turned behind the first K rows, it spills: 32.8 -> 38.0 and 67 -> 75.)
template <bool NARROW, typename T>
__device__ __forceinline__ void tile_ask_members(const TileCtx &t, const T *base, uint32_t RB, float4 (&rows)[4]) {
    const int row = max(t.member.x, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r)
        rows[r] = tile_row4<NARROW>(reinterpret_cast<const char *>(base) + ((uint32_t)lane_bcast(row, 4 * t.g + r) * RB + t.offv));
}

// Block after block, a block's loads ahead of its products.  Forms measured at L = 8192, k = 4 (1217 tiles of 4 blocks) and
// dropped: the rows of the next block loaded while one is used (a two-stage register pipeline: 47 us against 44, a wavefront
// per SIMD fewer; on few, tall tiles it was the better form until the parts of a tile came to be walked side by side, see
// tile_parts), groups of 32 rows (two member blocks per wavefront sharing the K / V
// registers: a third fewer rows through the L1s, two or three wavefronts per SIMD, 56 us; two wavefronts per head in step
// on the same entries, one member block each, so that the L1 fetches a row once: 60 us: the time follows the number
// of 16 x 16 blocks, 4716 against 6324, not the bytes), five or six wavefronts per SIMD by spilling (53 / 85 us).
template <typename Blk, typename Issue, typename Compute>
__device__ __forceinline__ void tile_walk(int nblk, Issue &&issue, Compute &&compute) {
    for (int b = 0; b < nblk; ++b) {
        Blk A;
        issue(A, b);
        issue_loads_first();
        compute(A);
        issue_loads_first();
    }
}

// The rows a block needs FIRST (the K rows of its scores) are asked for one block ahead, the others (V) when the block
// begins: sixteen more registers instead of the thirty-two of the two-stage pipeline, so four wavefronts per SIMD stay.
// once_loads_left(): called once the first loads have left, for work that waits for loads asked for before them.
template <typename Blk, typename IssueFirst, typename IssueRest, typename Compute, typename Hook>
__device__ __forceinline__ void tile_walk_first_ahead(int nblk, IssueFirst &&first, IssueRest &&rest, Compute &&compute, Hook &&once_loads_left) {
    Blk A, B;
    first(A, 0);
    issue_loads_first();
    once_loads_left();
    int b = 0;
    for (; b + 2 < nblk; b += 2) {
        rest(A, b);
        first(B, b + 1);
        issue_loads_first();
        compute(A);
        issue_loads_first();
        rest(B, b + 1);
        first(A, b + 2);
        issue_loads_first();
        compute(B);
        issue_loads_first();
    }
    rest(A, b);
    if (b + 1 < nblk) {
        first(B, b + 1);
        issue_loads_first();
        compute(A);
        issue_loads_first();
        rest(B, b + 1);
        issue_loads_first();
        compute(B);
    } else {
        issue_loads_first();
        compute(A);
    }
    issue_loads_first();
}

// Scores that are capped and lowered by distance (MOD): with u = scale (q.k + term),
//   s = cap tanh(u / cap) - slope[head] |pos[dst] - pos[src]|,   ds/du = 1 - tanh^2(u / cap),   dslope[head] = -sum over the pairs of dL/ds |pos - pos|
// A pair costs a handful of vector instructions more (tile_mod_scores), a block one load of its entries' positions by sixteen lanes, which
// travels with the block's rows and reaches the lanes through LDS, and nothing of an edge's size is read or written.
struct ScoreMod {
    float to_tanh, from_tanh;          // scale / cap, and cap in base-2 units; to_tanh 0: not capped
    float c[4], far;                   // tile_mod_scores: the polynomial's coefficients and bound for x^2
    float scale, slope_of;             // ... scale, and -scale / from_tanh^2
    const float *slopes;               // (heads), or null: no distance
    const float *pos_member, *pos_entry;       // positions of the plan's rows, of the rows its indices name
    float *part;                       // destination side: [group][head][part] sums of dL/ds |pos - pos|, or null
    float4 *split;                     // destination side: [slot][head] sums of p dP (float32 and with a score term: of ds before du), of p |pos - pos| and of
                                       // p over a split row's segment, or null
    bf16_t *low;                       // bfloat16 destination side: [slot][column] sums of p du K
};
struct NoMod {};
template <bool MOD> struct ModArg { typedef NoMod type; };
template <> struct ModArg<true> { typedef ScoreMod type; };

// What stands in rows that are not a member's neighbours must not reach its sums, and a product over a block's entries lets it: 0 x NaN.  So a wavefront whose
// sums (of any member) are not finite walks its tile once more (CAREFUL), with products that add the existing pairs alone and with every
// value of a pair that does not exist set to zero.  Rows that are finite, as nearly all are, cost this one look at the sums.
template <int N> __device__ __forceinline__ float tile_odd(const floatx4v (&acc)[N]) {         // 0, or NaN where something is infinite or NaN
    float x = 0.f;
#pragma unroll
    for (int nb = 0; nb < N; ++nb)
#pragma unroll
        for (int r = 0; r < 4; ++r) x = fmaf(acc[nb][r], 0.f, x);
    return x;
}
__device__ __forceinline__ bool tile_any_odd(float x) { return __builtin_amdgcn_ballot_w64(x != 0.f) != 0; }
template <bool ON> __device__ __forceinline__ float pair_if(int mask, int bit, float x) {        // x; with ON, 0 of a pair that does not exist
    if constexpr (ON) return where_pair_or_zero(mask, bit, x);
    else return x;
}
__device__ __forceinline__ float4 tile_four(const float4 &x) { return x; }
__device__ __forceinline__ float4 tile_four(const uint2 &x) {
    return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u));
}
// acc[nb][i] (member 4 g + i, column 4 c + nb) += w x rows over the pairs that exist; lane (c, g), register r: weight of member c with the entry whose
// columns 4 c .. 4 c + 3 it has and whose mask is mk[r]
template <typename Row> __device__ __forceinline__ void tile_axpy_pairs(const float (&w)[4], const int (&mk)[4], const Row (&rows)[4], int c, int g, floatx4v (&acc)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float4 mine = tile_four(rows[r]);
#pragma unroll 1
        for (int from = 0; from < 4; ++from) {
            const int at = 16 * from + c, mask = lane_bcast(mk[r], 16 * from);
            const float row[4] = {lane_bcast(mine.x, at), lane_bcast(mine.y, at), lane_bcast(mine.z, at), lane_bcast(mine.w, at)};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = lane_bcast(w[r], 16 * from + 4 * g + i);
#pragma unroll
                for (int nb = 0; nb < 4; ++nb) acc[nb][i] = (mask >> (4 * g + i)) & 1 ? fmaf(x, row[nb], acc[nb][i]) : acc[nb][i];
            }
        }
    }
}

// s (base-2 units) and scale ds/du of four pairs whose q.k (+ term) is x; pos_e: positions of the pairs' entries.
// |u / cap| <= 1/2, where nearly all scores lie (a score is a few units, a cap tens): tanh z = z + z w (c0 + c1 w + c2 w^2 + c3 w^3) with w = z^2,
// fitted by weighted least squares to the relative error, 1.5e-8; scale, cap and the change to base 2 sit in the coefficients, s = x (c + w' (...)) with w' = x^2,
// scale ds/du = scale - scale (s / cap)^2, and a wavefront without a larger score evaluates nothing else.  Beyond, (1 - e) / (1 + e) with
// e = exp(-2 |z|), whose difference keeps its digits there; for small z it is off by 2^-24 absolutely, which times a cap of 50 is more than all other
// roundings of a score.  The derivative is 4 e / (1 + e)^2 there: 1 - tanh^2 has lost half its digits at |z| = 4 and all of them at 9.  Below 2^-53 (|z| = 18.7)
// it counts as 0, as 1 - tanh^2 does in 64 bits.
__device__ __forceinline__ void tile_mod_scores(const ScoreMod &md, float scale_log2e, float slope_log2e, float pos_m, const float (&pos_e)[4],
                                                const float (&x)[4], float (&s)[4], float (&du)[4]) {
    if (md.to_tanh != 0.f) {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = x[r] * x[r];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[r] = x[r] * fmaf(fmaf(fmaf(fmaf(md.c[3], w[r], md.c[2]), w[r], md.c[1]), w[r], md.c[0]), w[r], scale_log2e);
            du[r] = fmaf(s[r] * s[r], md.slope_of, md.scale);
        }
        if (__builtin_amdgcn_ballot_w64(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])) > md.far) != 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(fabsf(x[r] * md.to_tanh) * (-2.f * LOG2E)), inv = __builtin_amdgcn_rcpf(1.f + e);
                s[r] = w[r] > md.far ? copysignf((1.f - e) * inv, x[r] * md.to_tanh) * md.from_tanh : s[r];
                du[r] = w[r] > md.far ? (e < 0x1p-55f ? 0.f : 4.f * e * inv * inv * md.scale) : du[r];
            }
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) { s[r] = x[r] * scale_log2e; du[r] = md.scale; }
    }
    if (md.slopes) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = fmaf(-slope_log2e, fabsf(pos_m - pos_e[r]), s[r]);
    }
}
// What the segments among the tile's members have summed up (lane (c, g), register r: columns 4 c .. 4 c + 3 of member 4 g + r), rounded, to md.low
template <int H, int D, bool NARROW> __device__ __forceinline__ void tile_store_low(const ScoreMod &md, const TileCtx &t, int r, const float4 &x, const Narrow &nw) {
    const int at = lane_bcast(tile_where(t.member), 4 * t.g + r);
    if (at >= -1 || (NARROW && 4 * t.c >= nw.d)) return;
    bf16_t *const to = md.low + (size_t)(-2 - at) * (NARROW ? nw.h * D : H * D) + t.head * D + (NARROW ? narrow_col(nw, t.c) : 4 * t.c);
    *reinterpret_cast<uintx2u *>(to) = uintx2u{pack_bf16(x.x, x.y), pack_bf16(x.z, x.w)};
}
template <int SP, int H, int D, bool NARROW>
__device__ __forceinline__ void tile_put_low(const ScoreMod &md, const TileCtx &t, float *mine, const float *part0, int stride, const floatx4v (&acc)[4], const Narrow &nw) {
    if constexpr (SP > 1) {
        constexpr int RS = 4 / SP;
        const float none[SP] = {};
        tile_park(mine, acc, t.lane);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RS; ++i) tile_store_low<H, D, NARROW>(md, t, t.part * RS + i, tile_meet<SP, false>(part0, stride, t.part * RS + i, t, none), nw);
        __syncthreads();
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) tile_store_low<H, D, NARROW>(md, t, r, make_float4(acc[0][r], acc[1][r], acc[2][r], acc[3][r]), nw);
    }
}
// sums of member c over the SP parts of a tile, in their order
template <int SP, int HW> __device__ __forceinline__ void tile_parts_sum(float4 (&meet)[HW][TILE_R], const TileCtx &t, float4 &sums) {
    if (t.g == 0) meet[t.wv][t.c] = sums;
    __syncthreads();
    sums = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < SP; ++i) {
        const float4 x = meet[i * (HW / SP) + t.wv % (HW / SP)][t.c];
        sums.x += x.x; sums.y += x.y; sums.z += x.z; sums.w += x.w;
    }
}
// The sum of a row's ds is zero, but for delta's rounding and the pairs', by which the row's mean distance multiplies: taken off slope_sum.  The rows of
// segments are left to k_score_split, where it runs.
template <int SP, int HW>
__device__ __forceinline__ void tile_slope_fix(const ScoreMod &md, const TileCtx &t, int heads, float ds_sum, float far_sum, float p_sum, float &slope_sum) {
    float4 sums = make_float4(groups_sum(ds_sum), groups_sum(far_sum), groups_sum(p_sum), 0.f);      // of member c, of this part
    if constexpr (SP > 1) {
        __shared__ float4 meet[HW][TILE_R];
        tile_parts_sum<SP, HW>(meet, t, sums);
    }
    const bool segment = t.member.y >= 0;
    if (!segment && sums.z != 0.f) slope_sum = fmaf(-sums.x / sums.z, far_sum, slope_sum);
    if (segment && md.split && t.g == 0 && t.part == 0) md.split[(size_t)t.member.y * heads + t.head] = sums;
}
// dslope of a wavefront's pairs (part s of SP of a group and head): the sum over its lanes
template <int SP> __device__ __forceinline__ void tile_put_slope_part(const ScoreMod &md, const TileCtx &t, int heads, float x) {
    if (!md.part) return;
    x = groups_sum(head_sum<16>(x));
    if (t.lane == 0) md.part[((size_t)t.grp * heads + t.head) * SP + t.part] = x;
}

template <typename T, int H, int D, int HW, bool DROP, int BIAS, bool NARROW = false, int SP = 1, bool MOD = false>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(4))) void k_attn_fwd_tile(
    bpt_plan P, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, T *__restrict__ o, float *__restrict__ lse,
    float *__restrict__ ws_acc, float *__restrict__ ws_ml, float scale_log2e, uint32_t drop_thr, uint32_t drop_seed, float drop_inv,
    const float *__restrict__ bias, Narrow nw, Keep keep, typename ModArg<MOD>::type md) {
    const int Hs = NARROW ? nw.h : H;                             // heads as lse, workspace and dropout keys count them
    const uint32_t RB = NARROW ? (uint32_t)(nw.heads * nw.d) * sizeof(T) : (uint32_t)(H * D * sizeof(T));        // bytes of a node row
    int block = (int)blockIdx.x;
    if constexpr (NARROW) block = keep_or_tile<HW * WAVE>(keep);
    if (NARROW && block < 0) return;
    T *const o_keep = NARROW ? reinterpret_cast<T *>(keep.o) : nullptr;
    TileCtx t;
    if (!tile_begin<T, H, D, HW, NARROW, SP>(P, t, nw, (unsigned)block)) return;
    __shared__ int2 ent_lds[HW][TILE_CHUNK];
    __shared__ int fst_lds[HW][BIAS == 2 ? TILE_CHUNK : 1];      // the entries' first pair numbers: where a term in pair order sits
    int2 *ent = ent_lds[t.wv];
    int *fst = BIAS == 2 ? fst_lds[t.wv] : nullptr;
    __shared__ __attribute__((aligned(16))) float kt_lds[HW][TILE_R * TILE_KT_STRIDE];
    float *kt = kt_lds[t.wv];
    __shared__ float pos_lds[HW][MOD ? TILE_R : 1];              // positions of the block's entries
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const char *kb = reinterpret_cast<const char *>(k), *vb = reinterpret_cast<const char *>(v);
    float qb[16];
    // The members' q rows are asked for behind the first block's K rows: asked for here, ahead of the loop, they are waited
    // for before the entry list is (one more round trip in front of the K rows).  They stay as they are and the scores are
    // scaled instead, so nothing has to happen to them between their arrival and the first product.
    const char *const qrow = reinterpret_cast<const char *>(q) + (size_t)max(t.member.x, 0) * RB + t.offa;
    // (with the score term the sixteen registers are not there; with dropout they just are, and it does not pay: L = 8192 level, 6 x 50
    // with dropout 97.7 -> 100 us)
    constexpr bool AHEAD = !DROP && BIAS == 0 && !MOD;
    if constexpr (!AHEAD) {
        float4 qr[4];
        tile_ask_members<NARROW>(t, q, RB, qr);
        tile_rows_to_operand<NARROW>(kt, qr, c, g, qb, nw);
    }
    float slope = 0.f, pos_m = 0.f;
    if constexpr (MOD) {
        if (md.slopes) {
            slope = md.slopes[t.head] * LOG2E;
            pos_m = md.pos_member[max(t.member.x, 0)];
        }
    }
    floatx4v acc[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
    float mref = m_init<MOD>(), lrun = 0.f;
    bool fresh = true;                                            // nothing has been summed up yet
    struct Blk {
        float4 kq[4];                                             // columns 4 c .. 4 c + 3 of the K rows of entries 4 r + g
        float4 vr[4];
        int mk[4], nv;                                            // bit c of mk[r]: the pair (entry 4 r + g, member c) exists; nv: entries of the block that exist
        int xe[DROP || BIAS == 1 ? 4 : 1];
        float bz[BIAS ? 4 : 1];
        float pos;                                                // of entry c, in the first lane group
    };
    auto walk = [&](auto again) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(again)::value;
    if constexpr (CAREFUL) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        if (p0 != t.p_begin) tile_ask_entries(P, p0, cnt, t.lane, er);
        tile_put_entries(er, ent, cnt, t.lane, fst);
        auto issue_k = [&](Blk &B, int b) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                B.kq[r] = tile_row4<NARROW>(kb + ((uint32_t)ent[TILE_R * b + 4 * r + g].x * RB + t.offv));
        };
        auto issue_rest = [&](Blk &B, int b) {
            if constexpr (DROP || BIAS == 1) tile_pair_eids(P, p0 + TILE_R * b + g, t.p_end, c, B.xe, 4);
            B.nv = min(TILE_R, cnt - TILE_R * b);
            if constexpr (MOD) {
                if (md.slopes && g == 0) B.pos = md.pos_entry[ent[TILE_R * b + c].x];
            }
            int idxv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int2 en = ent[TILE_R * b + 4 * r + g];
                idxv[r] = en.x; B.mk[r] = en.y;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                B.vr[r] = tile_row4<NARROW>(vb + ((uint32_t)idxv[r] * RB + t.offv));
            if constexpr (BIAS == 1) {
#pragma unroll
                for (int r = 0; r < 4; ++r) B.bz[r] = bias[tile_bias_at<H, 1>(P, t.head, B.xe[BIAS == 1 ? r : 0], 0)];
            }
            if constexpr (BIAS == 2) {
#pragma unroll
                for (int r = 0; r < 4; ++r) B.bz[r] = bias[tile_bias_at<H, 2>(P, t.head, 0, tile_pair_number(fst[TILE_R * b + 4 * r + g], B.mk[r], c))];
            }
        };
        auto compute = [&](const Blk &B) {
            float kr[16];
            if constexpr (MOD) {
                if (md.slopes && g == 0) pos_lds[t.wv][c] = B.pos;
            }
            tile_rows_to_operand<NARROW>(kt, B.kq, c, g, kr, nw);
            const floatx4v st = tile_dot(kr, qb);
            float sc[4];
            if constexpr (MOD) {
                float x[4], pos_e[4], du[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = BIAS ? st[r] + B.bz[BIAS ? r : 0] : st[r];
                    pos_e[r] = md.slopes ? pos_lds[t.wv][4 * r + g] : 0.f;
                }
                tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, sc, du);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[r] = where_pair(B.mk[r], c, sc[r]);
            } else
#pragma unroll
            for (int r = 0; r < 4; ++r)
                sc[r] = where_pair(B.mk[r], c, BIAS ? fmaf(st[r], scale_log2e, B.bz[BIAS ? r : 0] * scale_log2e) : st[r] * scale_log2e);
            const float mb = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
            if (__builtin_amdgcn_ballot_w64(mb > mref + MFMA_TAU) != 0) {
                const float mn = fmaxf(mref, groups_max(mb));    // over the four lanes of member c
                const float al = __builtin_amdgcn_exp2f(mref - mn);
                mref = mn;
                if (!fresh) {
                    lrun *= al;
                    // register r' of the accumulators belongs to member 4 g + r': its factor sits in lane 4 g + r'
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float a = lane_bcast(al, 4 * g + r);
#pragma unroll
                        for (int nb = 0; nb < 4; ++nb) acc[nb][r] *= a;
                    }
                }
            }
            fresh = false;
            float pr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pr[r] = __builtin_amdgcn_exp2f(sc[r] - mref);
                lrun += pr[r];                                   // the softmax denominator ignores dropout
                if constexpr (DROP)
                    pr[r] *= dropout_keep((uint32_t)B.xe[DROP ? r : 0] * (uint32_t)Hs + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
            }
            if constexpr (CAREFUL) tile_axpy_pairs(pr, B.mk, B.vr, c, g, acc);
            else tile_axpy_upto(pr, B.vr, acc, B.nv);
        };
        auto issue = [&](Blk &B, int b) { issue_k(B, b); issue_rest(B, b); };
        if constexpr (!AHEAD) tile_walk<Blk>(nblk, issue, compute);
        else tile_walk_first_ahead<Blk>(nblk, issue_k, issue_rest, compute, [&]() { if (p0 == t.p_begin) tile_load16<NARROW>(qrow, qb, g, nw); });
        wave_lds_fence();                                         // the piece is read to the end before the next one is staged
    }
    };
    walk(std::false_type{});
    if constexpr (MOD) {
        if (tile_any_odd(tile_odd(acc))) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
            mref = m_init<MOD>();
            lrun = 0.f;
            fresh = true;
            walk(std::true_type{});
        }
    }
    float lt = groups_sum(lrun);                                 // denominator of member c, in its four lanes
    if constexpr (SP > 1) {
        static_assert(TILE_PART_FWD_FLOATS <= TILE_R * TILE_KT_STRIDE, "a part fits its wavefront's piece");
        tile_meet_forward<SP, H, D, NARROW, MOD>(kt, kt_lds[t.wv % (HW / SP)], (HW / SP) * TILE_R * TILE_KT_STRIDE, t, acc, mref, lt, o, ws_acc, nw, o_keep);
        if (t.part != 0) return;
    } else {
        tile_store_rows<H, D, true, NARROW>(t, acc, has_sum<MOD>(lt) ? 1.f / lt : 0.f, o, ws_acc, nw, o_keep);
    }
    if (g == 0 && t.member.x >= 0) {                              // lanes 0 .. 15: one member each
        if (t.member.y < 0) {
            lse[(size_t)t.member.x * Hs + t.head] = has_sum<MOD>(lt) ? mref + log2f(lt) : 0.f;
        } else {
            ws_ml[((size_t)t.member.y * Hs + t.head) * 2] = mref;
            ws_ml[((size_t)t.member.y * Hs + t.head) * 2 + 1] = lt;
        }
    }
}

// Backward on tiles, destination side: per block the scores and dO . v of all 16 x 16 pairs (two products over the
// columns, the K and V rows turned in LDS from the layout they are loaded in), p = 2^(s - lse),
// ds = p (dO . v - delta) scale, dq += ds K (third product, on the K rows as loaded).  With dropout or a score term the
// kernel is compiled for three wavefronts per SIMD: at four it keeps the members' q rows in scratch memory and reads
// them back for every block (83 against 58 us with dropout at L = 8192, k = 4).
// (p, ds) of the pairs that exist go to a scratch in THIS side's order, compact:
// pds[head * n_edges + t] for the pair number t of (entry, member) = the entry's first pair + the rank of the member in
// its mask, so the lanes of an entry write one contiguous run and the runs of consecutive entries follow each other.  The
// source side looks its pairs up there through its pair mapping (grp_pairs = this side's pair numbers).  Writing in the
// source side's layout instead (scattered 8-byte stores here, contiguous reads there) cost this kernel a third of its
// time (126 against 85 us at L = 4096, k = 32); letting the source side recompute p and ds (two more products there,
// delta (n, H) handed over) measured slower than either on every graph tried.
template <typename T, int H, int D, int HW, bool DROP, int BIAS, bool NARROW = false, int SP = 1, bool MOD = false>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(DROP || BIAS || MOD ? 3 : 4))) void k_attn_bwd_dst_tile(
    bpt_plan P, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const T *__restrict__ o,
    const T *__restrict__ d_o, const float *__restrict__ lse, T *__restrict__ dq, float2 *__restrict__ pds, float *__restrict__ ws_dq,
    float scale, float scale_log2e, uint32_t drop_thr, uint32_t drop_seed, float drop_inv, const float *__restrict__ bias,
    float *__restrict__ ds_out, Narrow nw, typename ModArg<MOD>::type md) {
    const int Hs = NARROW ? nw.h : H;
    const uint32_t RB = NARROW ? (uint32_t)(nw.heads * nw.d) * sizeof(T) : (uint32_t)(H * D * sizeof(T));
    TileCtx t;
    if (!tile_begin<T, H, D, HW, NARROW, SP>(P, t, nw)) return;
    __shared__ int2 ent_lds[HW][TILE_CHUNK];
    __shared__ int fst_lds[HW][TILE_CHUNK];
    int2 *ent = ent_lds[t.wv];
    int *fst = fst_lds[t.wv];
    __shared__ __attribute__((aligned(16))) float kt_lds[HW][TILE_R * TILE_KT_STRIDE];
    float *kt = kt_lds[t.wv];
    __shared__ float pos_lds[HW][MOD ? TILE_R : 1];
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const char *kb = reinterpret_cast<const char *>(k), *vb = reinterpret_cast<const char *>(v);
    const size_t mrow = (size_t)max(t.member.x, 0) * RB + t.offa;
    float2 *const pds_h = pds + (size_t)t.head * (size_t)P.n_edges;     // this head's part of the scratch
    // the member's dO columns live in LDS (lane-major, read back before every product with them): with them in registers
    // the kernel needs 144 and a SIMD holds three wavefronts, without them 128 and four
    __shared__ floatx4v dob_lds[HW / SP][4][WAVE];
    floatx4v(&dob_h)[4][WAVE] = dob_lds[t.wv % (HW / SP)];
    // (q stays as it is and the scores are scaled, as in the forward: the same roundings in both)
    float qb[16], delta, lse_c;
    if constexpr (SP > 1) {
        // each part reads its 4 / SP steps of the members' rows for all of them
        __shared__ floatx4v q_lds[HW / SP][4][WAVE];
        __shared__ float delta_lds[HW][TILE_R];
        floatx4v(&q_h)[4][WAVE] = q_lds[t.wv % (HW / SP)];
        constexpr int TS = 4 / SP;
        floatx4v xq[TS], xd[TS], xo[TS];
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            const int at = t.part * TS + i;
            xq[i] = tile_load4<NARROW>(reinterpret_cast<const char *>(q) + mrow, at, g, nw);
            xd[i] = tile_load4<NARROW>(reinterpret_cast<const char *>(d_o) + mrow, at, g, nw);
            xo[i] = tile_load4<NARROW>(reinterpret_cast<const char *>(o) + mrow, at, g, nw);
        }
        lse_c = lse[(size_t)max(t.member.x, 0) * Hs + t.head];
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            q_h[t.part * TS + i][t.lane] = xq[i];
            dob_h[t.part * TS + i][t.lane] = xd[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) part = fmaf(xd[i][e], xo[i][e], part);
        }
        part = groups_sum(part);
        if (g == 0) delta_lds[t.wv][c] = part;
        __syncthreads();
        delta = 0.f;
#pragma unroll
        for (int i = 0; i < SP; ++i) delta += delta_lds[i * (HW / SP) + t.wv % (HW / SP)][c];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const floatx4v x = q_h[i][t.lane];
            qb[4 * i] = x[0]; qb[4 * i + 1] = x[1]; qb[4 * i + 2] = x[2]; qb[4 * i + 3] = x[3];
        }
    } else {
        float ob[16], dob[16];
        float4 qr[4], dr[4], orow[4];
        tile_ask_members<NARROW>(t, d_o, RB, dr);
        tile_ask_members<NARROW>(t, o, RB, orow);
        tile_ask_members<NARROW>(t, q, RB, qr);
        tile_rows_to_operand<NARROW>(kt, dr, c, g, dob, nw);
        tile_rows_to_operand<NARROW>(kt, orow, c, g, ob, nw);
        tile_rows_to_operand<NARROW>(kt, qr, c, g, qb, nw);
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) part = fmaf(dob[i], ob[i], part);
        delta = groups_sum(part);                                 // dO . O of member c, this head
        lse_c = lse[(size_t)max(t.member.x, 0) * Hs + t.head];
#pragma unroll
        for (int i = 0; i < 4; ++i) dob_h[i][t.lane] = floatx4v{dob[4 * i], dob[4 * i + 1], dob[4 * i + 2], dob[4 * i + 3]};
    }
    float slope = 0.f, pos_m = 0.f, slope_sum = 0.f, far_sum = 0.f, ds_sum = 0.f, p_sum = 0.f;
    if constexpr (MOD) {
        if (md.slopes) {
            slope = md.slopes[t.head] * LOG2E;
            pos_m = md.pos_member[max(t.member.x, 0)];
        }
    }
    floatx4v acc[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
    struct Blk {
        float4 kc[4], vc[4];                                      // columns 4 c .. 4 c + 3 of the K / V rows of entries 4 r + g
        int b, nv;                                                // which block of the piece; entries of it that exist
        int xe[DROP || BIAS == 1 ? 4 : 1];
        float bz[BIAS ? 4 : 1];
        float pos;                                                // of entry c, in the first lane group
    };
    auto walk = [&](auto again) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(again)::value;
    if constexpr (CAREFUL) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        if (p0 != t.p_begin) tile_ask_entries(P, p0, cnt, t.lane, er);
        tile_put_entries(er, ent, cnt, t.lane, fst);
        auto issue = [&](Blk &B, int b) {
            if constexpr (DROP || BIAS == 1) tile_pair_eids(P, p0 + TILE_R * b + g, t.p_end, c, B.xe, 4);
            B.b = b;
            if constexpr (MOD) {
                if (md.slopes && g == 0) B.pos = md.pos_entry[ent[TILE_R * b + c].x];
            }
            B.nv = min(TILE_R, cnt - TILE_R * b);
            int idxv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) idxv[r] = ent[TILE_R * b + 4 * r + g].x;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                B.kc[r] = tile_row4<NARROW>(kb + ((uint32_t)idxv[r] * RB + t.offv));
#pragma unroll
            for (int r = 0; r < 4; ++r)
                B.vc[r] = tile_row4<NARROW>(vb + ((uint32_t)idxv[r] * RB + t.offv));
            if constexpr (BIAS) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = TILE_R * b + 4 * r + g;
                    B.bz[r] = bias[tile_bias_at<H, BIAS>(P, t.head, B.xe[BIAS == 1 ? r : 0], BIAS == 2 ? tile_pair_number(fst[at], ent[at].y, c) : 0)];
                }
            }
        };
        auto compute = [&](const Blk &B) {
            int mask[4], number[4];                               // (read here, not kept from the block's issue on)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = TILE_R * B.b + 4 * r + g;
                mask[r] = ent[at].y;
                number[r] = tile_pair_number(fst[at], mask[r], c);
            }
            if constexpr (MOD) {
                if (md.slopes && g == 0) pos_lds[t.wv][c] = B.pos;
            }
            floatx4v st;
            {
                float kr[16];
                tile_rows_to_operand<NARROW>(kt, B.kc, c, g, kr, nw);
                st = tile_dot(kr, qb);
            }
            float va[16];
            tile_rows_to_operand<NARROW>(kt, B.vc, c, g, va, nw);
            float dob[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const floatx4v x = dob_h[i][t.lane];
                dob[4 * i] = x[0]; dob[4 * i + 1] = x[1]; dob[4 * i + 2] = x[2]; dob[4 * i + 3] = x[3];
            }
            const floatx4v dp = tile_dot(va, dob);
            float ds[4], sm[4], du[4], pos_e[4];
            if constexpr (MOD) {
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = BIAS ? st[r] + B.bz[BIAS ? r : 0] : st[r];
                    pos_e[r] = md.slopes ? pos_lds[t.wv][4 * r + g] : 0.f;
                }
                tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, sm, du);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float pe = where_pair_or_zero(mask[r], c, __builtin_amdgcn_exp2f((MOD ? sm[r] : BIAS ? fmaf(st[r], scale_log2e, B.bz[BIAS ? r : 0] * scale_log2e) : st[r] * scale_log2e) - lse_c));
                float mt = 1.f;                                   // dropout multiplier of this pair (as in the forward)
                if constexpr (DROP)
                    mt = dropout_keep((uint32_t)B.xe[DROP ? r : 0] * (uint32_t)Hs + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
                if constexpr (MOD) {
                    ds[r] = where_pair_or_zero(mask[r], c, pe * (dp[r] * mt - delta));
                    if (md.part) {
                        const float far = fabsf(pos_m - pos_e[r]);
                        slope_sum += pair_if<CAREFUL>(mask[r], c, ds[r] * far);
                        far_sum += pair_if<CAREFUL>(mask[r], c, pe * far);
                        ds_sum += pair_if<CAREFUL>(mask[r], c, ds[r]);
                        p_sum += pe;
                    }
                    ds[r] = pair_if<CAREFUL>(mask[r], c, ds[r] * du[r]);
                } else {
                    ds[r] = pe * (dp[r] * mt - delta) * scale;
                }
                pe *= mt;                                         // what multiplies v (forward) and dO (dV)
                if ((mask[r] >> c) & 1) {
                    pds_h[(uint32_t)number[r]] = make_float2(pe, ds[r]);
                    if constexpr (BIAS) ds_out[tile_bias_at<H, BIAS>(P, t.head, B.xe[BIAS == 1 ? r : 0], number[r])] = ds[r];   // dL/d(score before scaling)
                }
            }
            if constexpr (CAREFUL) tile_axpy_pairs(ds, mask, B.kc, c, g, acc);
            else tile_axpy_upto(ds, B.kc, acc, B.nv);
        };
        tile_walk<Blk>(nblk, issue, compute);
        wave_lds_fence();
    }
    };
    walk(std::false_type{});
    if constexpr (MOD) {
        if (tile_any_odd(tile_odd(acc) + (slope_sum + far_sum) * 0.f)) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
            slope_sum = far_sum = ds_sum = p_sum = 0.f;
            walk(std::true_type{});
        }
    }
    if constexpr (MOD) {
        if (md.part) tile_slope_fix<SP, HW>(md, t, Hs, ds_sum, far_sum, p_sum, slope_sum);
        tile_put_slope_part<SP>(md, t, Hs, slope_sum);
    }
    if constexpr (SP > 1) {
        tile_park(kt, acc, t.lane);
        __syncthreads();
        tile_meet_and_store<SP, H, D, NARROW>(kt_lds[t.wv % (HW / SP)], (HW / SP) * TILE_R * TILE_KT_STRIDE, t, dq, ws_dq, nw);
    } else {
        tile_store_rows<H, D, false, NARROW>(t, acc, 1.f, dq, ws_dq, nw);
    }
}

// Backward on tiles, source side (groups of the out-CSR plan: members = source rows, entries = destinations):
// dk += ds^T q, dv += p^T dO with (p, ds) of every pair fetched from the scratch the destination side filled, at the
// destination side's pair number that this plan's grp_pairs gives for (entry, member).
//
// A lane asks for the pairs of ONE entry (destination) with four neighbouring members, not of one member with four entries:
// the destination side numbers the pairs of a tile by its entries, which are this side's members, so lanes c, the
// destinations of a block, mostly read one run of 8 bytes each per member instead of 16 places 8 bytes x (members per entry)
// apart, and the four positions are one load.  The block of (p, ds) is turned in LDS on the way into the products, which also
// frees its registers: the next block's (p, ds) are asked for behind this block's rows and the positions of the one after that,
// so neither is waited for, in 117 registers (two sets of (p, ds) in registers: 128 and 44 bytes spilled, 89 -> 100 us for the
// 32-graph batch).  The first positions leave with the entry list.  8 heads, before -> now: L = 32768, k = 4 218 -> 210 us;
// L = 4096, k = 32 54.1 -> 52.2; window 128 27.2 -> 25.6 (before: rows read a block ahead at three wavefronts per SIMD, which is
// not needed any more); 6 heads of 50 columns 68.5 -> 65.6; 32-graph batch and L = 8192, k = 4 level.
constexpr int TILE_WT_STRIDE = 18;                                // float2 per entry: 16 members + 2 (writes and reads spread over the banks)
typedef int intx4u __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ void tile_pair_positions(const bpt_plan &P, int entry, int g, int (&pos)[4]) {
    const intx4u x = *reinterpret_cast<const intx4u *>(P.grp_pairs + (size_t)entry * TILE_R + 4 * g);
    pos[0] = x[0]; pos[1] = x[1]; pos[2] = x[2]; pos[3] = x[3];
}
template <typename T, int H, int D, int HW, bool NARROW = false, int SP = 1, bool MOD = false>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(4))) void k_attn_bwd_src_tile(
    bpt_plan P, const T *__restrict__ q, const T *__restrict__ d_o, const float2 *__restrict__ pds, T *__restrict__ dk, T *__restrict__ dv,
    float *__restrict__ ws_dk, float *__restrict__ ws_dv, Narrow nw) {
    const uint32_t RB = NARROW ? (uint32_t)(nw.heads * nw.d) * sizeof(T) : (uint32_t)(H * D * sizeof(T));
    TileCtx t;
    if (!tile_begin<T, H, D, HW, NARROW, SP>(P, t, nw)) return;
    // a wavefront's piece: its entry list and its block of (p, ds), afterwards (SP > 1) what it has summed up
    constexpr int ENT = TILE_CHUNK * 2, LIVE = ENT + TILE_R * TILE_WT_STRIDE * 2, PIECE = SP > 1 ? 2 * TILE_PART_FLOATS : LIVE;
    static_assert(PIECE >= LIVE, "the lists fit");
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    int2 *ent = reinterpret_cast<int2 *>(piece[t.wv]);
    float2 *const wt = reinterpret_cast<float2 *>(piece[t.wv] + ENT);
    const int c = t.c, g = t.g;
    const char *qb = reinterpret_cast<const char *>(q), *db = reinterpret_cast<const char *>(d_o);
    const float2 *const pds_h = pds + (size_t)t.head * (size_t)P.n_edges;
    floatx4v ak[4], av[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) { ak[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; av[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
    // Both products contract over the block's entries, four per step; lane group g takes entries 4 r + g in step r, so that
    // the steps past the end of the group's list (half of a group's last block on average) can be left out.
    struct Blk {
        float4 qr[4], dr[4];
        int mk[4], nv;                                            // bit c of mk[r]: the pair (entry 4 r + g, member c) exists; nv: entries of the block that exist
    };
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    int pos[4];
    float2 w[4];                                                  // (p, ds) of the pairs (entry c, member 4 g + r) of the next block
    auto positions = [&](int first_entry) { tile_pair_positions(P, min(first_entry + c, t.p_end - 1), g, pos); };
    if (t.p_end > t.p_begin) positions(t.p_begin);
    issue_loads_first();
    auto walk = [&](auto again) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(again)::value;
    if constexpr (CAREFUL) {
        tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
        positions(t.p_begin);
    }
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        if (p0 != t.p_begin) tile_ask_entries(P, p0, cnt, t.lane, er);
        tile_put_entries(er, ent, cnt, t.lane);
        if (p0 == t.p_begin) {
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = pds_h[(uint32_t)pos[r]];
            positions(p0 + TILE_R);
        }
        auto put_pairs = [&]() {
            floatx4v *const wp = reinterpret_cast<floatx4v *>(wt + c * TILE_WT_STRIDE + 4 * g);
            wp[0] = floatx4v{w[0].x, w[0].y, w[1].x, w[1].y};
            wp[1] = floatx4v{w[2].x, w[2].y, w[3].x, w[3].y};
            wave_lds_fence();
        };
        auto issue_rows = [&](Blk &B, int b) {
            B.nv = min(TILE_R, cnt - TILE_R * b);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int2 en = ent[TILE_R * b + 4 * r + g];
                B.mk[r] = en.y;
                const uint32_t off = (uint32_t)en.x * RB + t.offv;
                B.qr[r] = tile_row4<NARROW>(qb + off);
                B.dr[r] = tile_row4<NARROW>(db + off);
            }
        };
        auto compute = [&](const Blk &B) {
            float pe[4], ds[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float2 w = wt[(4 * r + g) * TILE_WT_STRIDE + c];
                pe[r] = where_pair_or_zero(B.mk[r], c, w.x);      // the scratch of pairs that do not exist is not initialised
                ds[r] = where_pair_or_zero(B.mk[r], c, w.y);
            }
            wave_lds_fence();                                     // (read before the next block's are written)
            if constexpr (CAREFUL) {
                tile_axpy_pairs(ds, B.mk, B.qr, c, g, ak);
                tile_axpy_pairs(pe, B.mk, B.dr, c, g, av);
            } else {
                tile_axpy_upto(ds, B.qr, ak, B.nv);
                tile_axpy_upto(pe, B.dr, av, B.nv);
            }
        };
        for (int b = 0; b < nblk; ++b) {
            Blk B;
            issue_rows(B, b);
            issue_loads_first();
            put_pairs();
            if (p0 + TILE_R * (b + 1) < t.p_end) {
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = pds_h[(uint32_t)pos[r]];
                positions(p0 + TILE_R * (b + 2));
            }
            issue_loads_first();
            compute(B);
            issue_loads_first();
        }
        wave_lds_fence();
    }
    };
    walk(std::false_type{});
    if constexpr (MOD) {
        if (tile_any_odd(tile_odd(ak) + tile_odd(av))) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) { ak[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; av[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
            walk(std::true_type{});
        }
    }
    if constexpr (SP > 1) {
        constexpr int NEXT = (HW / SP) * PIECE;
        tile_park(piece[t.wv], ak, t.lane);
        tile_park(piece[t.wv] + TILE_PART_FLOATS, av, t.lane);
        __syncthreads();
        const float *const part0 = piece[t.wv % (HW / SP)];
        tile_meet_and_store<SP, H, D, NARROW>(part0, NEXT, t, dk, ws_dk, nw);
        tile_meet_and_store<SP, H, D, NARROW>(part0 + TILE_PART_FLOATS, NEXT, t, dv, ws_dv, nw);
    } else {
        tile_store_rows<H, D, false, NARROW>(t, ak, 1.f, dk, ws_dk, nw);
        tile_store_rows<H, D, false, NARROW>(t, av, 1.f, dv, ws_dv, nw);
    }
}

// ---- Dense tiles for bfloat16 rows.  Same walk and the same lane roles as the float32 tile kernels above, on
// v_mfma_f32_16x16x32_bf16 (products over the 64 columns: two instructions) and v_mfma_f32_16x16x16_bf16 (products over
// the 16 entries of a block: one instruction per four output columns), float32 accumulation:
//   lane (c, g) holds columns 16 g .. 16 g + 15 of the row of entry c (32 contiguous bytes; slot j of step t of the product
//   stands for column 16 g + 8 t + j in both operands).
// Heads of 64 columns: rows go through LDS for both kinds of product (k_attn_fwd_rows_bf16, k_attn_bwd_dst_rows_bf16,
// k_attn_bwd_src_tile_bf16_again; tile_ask_rows_bf16 says why), the next block's asked for while this one's are used.  Narrower heads, and
// the source side that reads (p, ds) back: a lane loads columns 4 c .. 4 c + 3 of the rows of entries 4 g + r (8 bytes; the B
// operand of output columns {4 c + nb} takes element nb of each of the four, packed by byte permutes), and the entries' rows
// are turned in LDS for the products over the columns (tile_rows_to_operand_bf16).
// Probabilities and ds are rounded to bfloat16 where they enter a product (the softmax denominator is summed unrounded);
// the scratch between the two backward kernels, where there is one, holds (p, ds) as two bfloat16 in 4 bytes, by head and destination-side pair number.
constexpr int TILE_BF16_WPE = 5, TILE_BF16_WPE_DST = 5, TILE_BF16_WPE_SRC = 5, TILE_BF16_WPE_AGAIN = 4;     // wavefronts per SIMD the bfloat16 tile kernels are compiled for
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef short shortx4v __attribute__((ext_vector_type(4)));
union Bf8 { bf16x8v v; uint4 q; };
union Bf4 { shortx4v v; uint32_t u[2]; };

__device__ __forceinline__ uint32_t pack_lo16(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }   // (a.lo, b.lo)
__device__ __forceinline__ uint32_t pack_hi16(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }   // (a.hi, b.hi)

// B operand of output columns {4 c + nb}: element nb of the 8-byte pieces of the rows of entries 4 g + r, r = 0 .. 3
template <int NB>
__device__ __forceinline__ Bf4 tile_cols_bf16(const uint2 (&rows)[4]) {
    Bf4 b;
    if constexpr (NB == 0) { b.u[0] = pack_lo16(rows[0].x, rows[1].x); b.u[1] = pack_lo16(rows[2].x, rows[3].x); }
    if constexpr (NB == 1) { b.u[0] = pack_hi16(rows[0].x, rows[1].x); b.u[1] = pack_hi16(rows[2].x, rows[3].x); }
    if constexpr (NB == 2) { b.u[0] = pack_lo16(rows[0].y, rows[1].y); b.u[1] = pack_lo16(rows[2].y, rows[3].y); }
    if constexpr (NB == 3) { b.u[0] = pack_hi16(rows[0].y, rows[1].y); b.u[1] = pack_hi16(rows[2].y, rows[3].y); }
    return b;
}
// acc[nb][r'] (member 4 g + r', column 4 c + nb) += sum over the block's entries of w[member c][entry 4 g + r] * row[entry][column]
__device__ __forceinline__ void tile_axpy_bf16(const Bf4 &w, const uint2 (&rows)[4], floatx4v (&acc)[4]) {
    acc[0] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(w.v, tile_cols_bf16<0>(rows).v, acc[0], 0, 0, 0);
    acc[1] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(w.v, tile_cols_bf16<1>(rows).v, acc[1], 0, 0, 0);
    acc[2] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(w.v, tile_cols_bf16<2>(rows).v, acc[2], 0, 0, 0);
    acc[3] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(w.v, tile_cols_bf16<3>(rows).v, acc[3], 0, 0, 0);
}
// register r of lane (c, g) = sum over the 64 columns of a[entry 4 g + r] * b[member c]
__device__ __forceinline__ floatx4v tile_dot_bf16(const Bf8 (&a)[2], const Bf8 (&b)[2]) {
    floatx4v s = floatx4v{0.f, 0.f, 0.f, 0.f};
    s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0].v, b[0].v, s, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1].v, b[1].v, s, 0, 0, 0);
}
__device__ __forceinline__ void tile_load_row_bf16(const char *p, Bf8 (&out)[2], int g, const Narrow &nw) {
    uint32_t w[8];
#pragma unroll
    for (int t = 0; t < 4; ++t) {                                 // quad 4 g + t; d is even, so a quad is shifted by whole words
        const int quad = 4 * (4 * g + t), col = min(quad, nw.d - 4);
        const uintx2u x = *reinterpret_cast<const uintx2u *>(p + 2 * col);
        w[2 * t] = col >= quad ? x[0] : 0u;
        w[2 * t + 1] = col + 2 >= quad ? x[1] : 0u;
    }
    out[0].q = make_uint4(w[0], w[1], w[2], w[3]);
    out[1].q = make_uint4(w[4], w[5], w[6], w[7]);
}
template <bool NARROW> __device__ __forceinline__ uint2 tile_row4_bf16(const char *p) {
    if constexpr (NARROW) {
        const uintx2u x = *reinterpret_cast<const uintx2u *>(p);
        return make_uint2(x[0], x[1]);
    } else {
        return *reinterpret_cast<const uint2 *>(p);
    }
}
// As tile_rows_to_operand: the rows of a block's entries, loaded as columns 4 c .. 4 c + 3 of the rows of entries 4 g + r
// (the sixteen lanes of a lane group read one row's 128 contiguous bytes), turned in a wavefront-private piece of LDS
// into the operand of the products over the columns (lane (c, g): columns 16 g .. 16 g + 15 of the row of entry c).
// Rows of TILE_KT_BYTES_BF16 = 128 + 16 bytes: the sixteen rows of a read fall on different banks.
constexpr int TILE_KT_BYTES_BF16 = 144;
typedef uint32_t uintx4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void tile_rows_to_operand_bf16(char *kt, const uint2 (&rows)[4], int c, int g, Bf8 (&out)[2], const Narrow &nw) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
        *reinterpret_cast<uintx2v *>(kt + (4 * g + r) * TILE_KT_BYTES_BF16 + 8 * c) =           // (d is even: words are whole)
            uintx2v{narrow_again<true>(nw, c, 0) ? 0u : rows[r].x, narrow_again<true>(nw, c, 2) ? 0u : rows[r].y};
    wave_lds_fence();
    const char *src = kt + c * TILE_KT_BYTES_BF16 + 32 * g;
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
        const uintx4v x = *reinterpret_cast<const uintx4v *>(src + 16 * h2);
        out[h2].q = make_uint4(x[0], x[1], x[2], x[3]);
    }
    wave_lds_fence();                                             // (read before the next block's rows are written)
}

constexpr int TILE_KT_FLOATS_BF16 = TILE_R * TILE_KT_BYTES_BF16 / 4;
// Rows of 64 columns, 16 bytes a lane: lane l asks for piece l % 8 of rows l / 8 and 8 + l / 8 of sixteen, puts them into LDS as
// above, and both kinds of product read them there: the products over the columns the row of entry c, the sums over the
// entries their columns, transposed (tile_axpy_rows_bf16), so that the registers are free for the next block's rows.
//
// What bounds the bfloat16 kernels is the texture addresser, which takes a vector memory instruction four lanes at a time: 16 cycles
// for one whose neighbouring lanes read on in a line, whatever a lane reads of it, 64 where each lane's line is another
// (by that count 614 k of the source side's 750 k cycles at 16 heads, L = 32768, k = 8; 250 k now).  Rows of eight bytes a lane took twice the instructions, members' rows
// read row by lane four times the cycles, (lse, delta) of a block's entries read by all 64 lanes as many as its rows.  So: rows, members'
// rows and results in 16 bytes a lane, along the rows; single words of a row by one lane group.  Nothing else helped the source side there:
// its rows a block ahead through LDS but 8 bytes a lane 333 -> 343 us; 16 bytes a lane 315; the members and (lse, delta) too 303;
// free of bank conflicts in LDS 281 to 290.  Kernels before -> after, forward / destination / source side: 16 heads at L = 32768, k = 8 184 / 240 / 333
// -> 162 / 208 / 285 us, 8 heads at L = 8192, k = 4 17.1 / 24.6 / 26.5 -> 16.4 / 22.8 / 23.6.  Training passes: window of 64 at L = 16384,
// 16 heads 163.5 -> 139.8, 32-graph batch 152 -> 139.8, L = 16384, k = 8 180 -> 158, with dropout at L = 32768, k = 8 818 -> 760.
__device__ __forceinline__ void tile_ask_rows_bf16(const char *base, const uint32_t (&off)[2], uintx4v (&rows)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) rows[r] = *reinterpret_cast<const uintx4v *>(base + off[r]);
}
// In LDS such rows lie 128 bytes apart, piece j of row e at place j ^ piece_turn(e): two rows of a write, the sixteen rows of an operand's
// read and the eight rows of a transposed read (32 lanes of 8 bytes, two pieces a row) fall on different banks.
constexpr int TILE_ROWS_FLOATS_BF16 = TILE_R * 32;
__device__ __forceinline__ int piece_turn(int e) { return (e & 6) | (e >> 3); }
__device__ __forceinline__ void tile_put_rows_bf16(char *kt, const uintx4v (&rows)[2], int lane) {
    const int at = (lane >> 3) * 128 + 16 * ((lane & 7) ^ piece_turn(lane >> 3));
    *reinterpret_cast<uintx4v *>(kt + at) = rows[0];
    *reinterpret_cast<uintx4v *>(kt + (at ^ 16) + 1024) = rows[1];
}
__device__ __forceinline__ void tile_operand_bf16(const char *kt, int c, int g, Bf8 (&out)[2]) {
    const int at = c * 128 + 16 * ((2 * g) ^ piece_turn(c));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uintx4v x = *reinterpret_cast<const uintx4v *>(kt + (at ^ (16 * i)));
        out[i].q = make_uint4(x[0], x[1], x[2], x[3]);
    }
}
// byte offsets of this lane's pieces of the members' rows / of the rows of the sixteen entries at `ent`
__device__ __forceinline__ uint32_t tile_piece_at(const TileCtx &t) { return (uint32_t)(t.head * 128 + 16 * (t.lane & 7)); }
template <uint32_t RB> __device__ __forceinline__ void tile_member_offsets(const TileCtx &t, uint32_t (&off)[2]) {
    const int row = max(t.member.x, 0);
#pragma unroll
    for (int r = 0; r < 2; ++r) off[r] = (uint32_t)lane_bcast(row, 8 * r + (t.lane >> 3)) * RB + tile_piece_at(t);
}
template <uint32_t RB> __device__ __forceinline__ void tile_entry_offsets(const TileCtx &t, const int2 *ent, uint32_t (&off)[2]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) off[r] = (uint32_t)ent[8 * r + (t.lane >> 3)].x * RB + tile_piece_at(t);
}
// masks of entries 4 g .. 4 g + 3
__device__ __forceinline__ void tile_masks(const int2 *ent, int g, int (&mk)[4]) {
    const int4 e01 = *reinterpret_cast<const int4 *>(&ent[4 * g]), e23 = *reinterpret_cast<const int4 *>(&ent[4 * g + 2]);
    mk[0] = e01.y; mk[1] = e01.w; mk[2] = e23.y; mk[3] = e23.w;
}
// acc += w^T rows, by column: lane (c, g), register r of acc[nb] = column 16 nb + 4 g + r of member c
__device__ __forceinline__ void tile_axpy_rows_bf16(const Bf4 &w, const char *kt, int c, int g, floatx4v (&acc)[4]) {
    // sixteen lanes read four rows of sixteen columns and are given one column of the four each
    const int e = 4 * g + (c >> 2), at = e * 128 + 16 * (((c >> 1) & 1) ^ piece_turn(e)) + 8 * (c & 1);
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
        const shortx4v cols = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4v *)(kt + (at ^ (32 * nb))));
        acc[nb] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(cols, w.v, acc[nb], 0, 0, 0);
    }
}
// ... over the pairs that exist (tile_odd), lane (c, g), register r of w and mk: entry 4 g + r
__device__ __forceinline__ void tile_axpy_pairs_bf16(const float (&w)[4], const int (&mk)[4], const char *kt, int c, int g, floatx4v (&acc)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll 1
        for (int from = 0; from < 4; ++from) {
            const int e = 4 * from + r, at = e * 128 + 16 * ((g >> 1) ^ piece_turn(e)) + 8 * (g & 1), mask = lane_bcast(mk[r], 16 * from);
            const float x = lane_bcast(w[r], 16 * from + c);
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) {
                const float4 row = tile_four(*reinterpret_cast<const uint2 *>(kt + (at ^ (32 * nb))));
                const float cols[4] = {row.x, row.y, row.z, row.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[nb][i] = (mask >> c) & 1 ? fmaf(x, cols[i], acc[nb][i]) : acc[nb][i];
            }
        }
}
// Such sums through LDS (TILE_R * TILE_TURN_STRIDE floats): into the tile kernels' other order (lane (c, g), register r: columns 4 c .. 4 c + 3
// of member 4 g + r), or to where the members' rows go.
constexpr int TILE_TURN_STRIDE = 68;
__device__ __forceinline__ void tile_put_sums(float *sh, const floatx4v (&acc)[4], int c, int g) {
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) *reinterpret_cast<floatx4v *>(sh + c * TILE_TURN_STRIDE + 16 * nb + 4 * g) = acc[nb];
    wave_lds_fence();
}
__device__ __forceinline__ void tile_sums_by_row(float *sh, floatx4v (&acc)[4], int c, int g) {
    tile_put_sums(sh, acc, c, g);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const floatx4v x = *reinterpret_cast<const floatx4v *>(sh + (4 * g + r) * TILE_TURN_STRIDE + 4 * c);
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) acc[nb][r] = x[nb];
    }
    wave_lds_fence();
}
template <int H, int D>
__device__ __forceinline__ void tile_store_sums(const TileCtx &t, float *sh, const floatx4v (&acc)[4], bf16_t *__restrict__ out, float *__restrict__ ws) {
    tile_put_sums(sh, acc, t.c, t.g);
    const int where = tile_where(t.member);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int m = 8 * r + (t.lane >> 3), at = lane_bcast(where, m);
        const floatx4v *const from = reinterpret_cast<const floatx4v *>(sh + m * TILE_TURN_STRIDE + 8 * (t.lane & 7));
        const floatx4v x = from[0], y = from[1];
        if (at >= 0) {                                            // (node tensors end before 4 GiB)
            char *const to = reinterpret_cast<char *>(out) + ((uint32_t)at * (uint32_t)(H * D * 2) + tile_piece_at(t));
            __builtin_nontemporal_store(uintx4v{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3])},
                                        reinterpret_cast<uintx4v *>(to));
        } else if (at < -1) {
            floatx4v *const to = reinterpret_cast<floatx4v *>(ws + (size_t)(-2 - at) * (H * D) + t.head * D + 8 * (t.lane & 7));
            to[0] = x;
            to[1] = y;
        }
    }
    wave_lds_fence();
}

template <int H, int D, int HW, int WPE, bool DROP, int BIAS, int SP, bool MOD = false>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(DROP || BIAS || MOD ? WPE - 1 : WPE))) void k_attn_fwd_rows_bf16(
    bpt_plan P, const bf16_t *__restrict__ q, const bf16_t *__restrict__ k, const bf16_t *__restrict__ v, bf16_t *__restrict__ o,
    float *__restrict__ lse, float *__restrict__ ws_acc, float *__restrict__ ws_ml, float scale_log2e, uint32_t drop_thr,
    uint32_t drop_seed, float drop_inv, const float *__restrict__ bias, typename ModArg<MOD>::type md) {
    constexpr uint32_t RB = H * D * 2;
    const Narrow nw{};
    TileCtx t;
    if (!tile_begin<bf16_t, H, D, HW, false, SP>(P, t, nw)) return;
    __shared__ int2 ent_lds[HW][TILE_CHUNK];
    __shared__ int fst_lds[HW][BIAS == 2 ? TILE_CHUNK : 1];      // the entries' first pair numbers: where a term in pair order sits
    int2 *ent = ent_lds[t.wv];
    int *fst = BIAS == 2 ? fst_lds[t.wv] : nullptr;
    constexpr int PIECE = 2 * TILE_ROWS_FLOATS_BF16 + 4 * TILE_R;      // (the turned sums' rows are longer)
    static_assert(PIECE >= TILE_PART_FWD_FLOATS && PIECE >= TILE_R * TILE_TURN_STRIDE, "parts and turned sums fit the rows' piece");
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    __shared__ __attribute__((aligned(16))) float pos_lds[HW][MOD ? TILE_R : 4];      // positions of the block's entries
    char *const k_lds = reinterpret_cast<char *>(piece[t.wv]), *const v_lds = k_lds + 4 * TILE_ROWS_FLOATS_BF16;
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const char *kb = reinterpret_cast<const char *>(k), *vb = reinterpret_cast<const char *>(v);
    uintx4v qr[2];
    {
        uint32_t off[2];
        tile_member_offsets<RB>(t, off);
        tile_ask_rows_bf16(reinterpret_cast<const char *>(q), off, qr);
    }
    issue_loads_first();
    Bf8 qb[2];
    float slope = 0.f, pos_m = 0.f;
    if constexpr (MOD) {
        if (md.slopes) {
            slope = md.slopes[t.head] * LOG2E;
            pos_m = md.pos_member[max(t.member.x, 0)];
        }
    }
    floatx4v acc[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
    float mref = m_init<MOD>(), lrun = 0.f;
    bool fresh = true;                                            // nothing has been summed up yet
    struct Blk {
        uintx4v kr[2], vr[2];
        int xe[DROP || BIAS == 1 ? 4 : 1];
        float bz[BIAS ? 4 : 1];
        float pos;                                                // of entry c, in the first lane group
    };
    auto walk = [&](auto again) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(again)::value;
    if constexpr (CAREFUL) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        if (p0 != t.p_begin) tile_ask_entries(P, p0, cnt, t.lane, er);
        tile_put_entries(er, ent, cnt, t.lane, fst);
        auto issue = [&](Blk &B, int b) {
            if constexpr (DROP || BIAS == 1) tile_pair_eids(P, p0 + TILE_R * b + 4 * g, t.p_end, c, B.xe);
            if constexpr (MOD) {
                if (md.slopes && g == 0) B.pos = md.pos_entry[ent[TILE_R * b + c].x];
            }
            uint32_t off[2];
            tile_entry_offsets<RB>(t, ent + TILE_R * b, off);
            tile_ask_rows_bf16(kb, off, B.kr);
            tile_ask_rows_bf16(vb, off, B.vr);
            if constexpr (BIAS == 1) {
#pragma unroll
                for (int r = 0; r < 4; ++r) B.bz[r] = bias[tile_bias_at<H, 1>(P, t.head, B.xe[BIAS == 1 ? r : 0], 0)];
            }
            if constexpr (BIAS == 2) {
                int mk[4];
                tile_masks(ent + TILE_R * b, g, mk);
#pragma unroll
                for (int r = 0; r < 4; ++r) B.bz[r] = bias[tile_bias_at<H, 2>(P, t.head, 0, tile_pair_number(fst[TILE_R * b + 4 * g + r], mk[r], c))];
            }
        };
        Blk B;
        issue(B, 0);
        issue_loads_first();
        if (!CAREFUL && p0 == t.p_begin) {
            tile_put_rows_bf16(k_lds, qr, t.lane);
            wave_lds_fence();
            tile_operand_bf16(k_lds, c, g, qb);
            wave_lds_fence();
        }
        for (int b = 0; b < nblk; ++b) {
            int mk[4], xe[DROP ? 4 : 1];
            float bz[BIAS ? 4 : 1];
            tile_masks(ent + TILE_R * b, g, mk);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (DROP) xe[DROP ? r : 0] = B.xe[DROP ? r : 0];
                if constexpr (BIAS) bz[BIAS ? r : 0] = B.bz[BIAS ? r : 0];
            }
            tile_put_rows_bf16(k_lds, B.kr, t.lane);
            tile_put_rows_bf16(v_lds, B.vr, t.lane);
            if constexpr (MOD) {
                if (md.slopes && g == 0) pos_lds[t.wv][c] = B.pos;
            }
            wave_lds_fence();
            if (b + 1 < nblk) issue(B, b + 1);
            issue_loads_first();
            Bf8 kr[2];
            tile_operand_bf16(k_lds, c, g, kr);
            const floatx4v st = tile_dot_bf16(kr, qb);
            float sc[4];
            if constexpr (MOD) {
                float x[4], du[4];
                const floatx4v pe = *reinterpret_cast<const floatx4v *>(&pos_lds[t.wv][4 * g]);
                const float pos_e[4] = {pe[0], pe[1], pe[2], pe[3]};
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = BIAS ? st[r] + bz[BIAS ? r : 0] : st[r];
                tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, sc, du);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[r] = where_pair(mk[r], c, sc[r]);
            } else
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[r] = where_pair(mk[r], c, (BIAS ? st[r] + bz[BIAS ? r : 0] : st[r]) * scale_log2e);
            const float mb = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
            if (__builtin_amdgcn_ballot_w64(mb > mref + MFMA_TAU) != 0) {
                const float mn = fmaxf(mref, groups_max(mb));    // over the four lanes of member c
                const float al = __builtin_amdgcn_exp2f(mref - mn);
                mref = mn;
                if (!fresh) {
                    lrun *= al;
#pragma unroll
                    for (int nb = 0; nb < 4; ++nb) acc[nb] *= al;
                }
            }
            fresh = false;
            float pr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pr[r] = __builtin_amdgcn_exp2f(sc[r] - mref);
                lrun += pr[r];                                   // the softmax denominator ignores dropout
                if constexpr (DROP)
                    pr[r] *= dropout_keep((uint32_t)xe[DROP ? r : 0] * (uint32_t)H + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
            }
            if constexpr (CAREFUL) {
                tile_axpy_pairs_bf16(pr, mk, v_lds, c, g, acc);
            } else {
                Bf4 pa;
                pa.u[0] = pack_bf16(pr[0], pr[1]);
                pa.u[1] = pack_bf16(pr[2], pr[3]);
                tile_axpy_rows_bf16(pa, v_lds, c, g, acc);
            }
            wave_lds_fence();                                     // (read before the next block's are written)
            issue_loads_first();
        }
    }
    };
    walk(std::false_type{});
    if constexpr (MOD) {
        if (tile_any_odd(tile_odd(acc))) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
            mref = m_init<MOD>();
            lrun = 0.f;
            fresh = true;
            walk(std::true_type{});
        }
    }
    float lt = groups_sum(lrun);
    if constexpr (SP > 1) {
        tile_sums_by_row(piece[t.wv], acc, c, g);
        tile_meet_forward<SP, H, D, false, MOD>(piece[t.wv], piece[t.wv % (HW / SP)], (HW / SP) * PIECE, t, acc, mref, lt, o, ws_acc, nw, static_cast<bf16_t *>(nullptr));
        if (t.part != 0) return;
    } else {
        if (t.member.y < 0) {                                     // (segments of a split row are stored as summed up)
            const float inv = has_sum<MOD>(lt) ? 1.f / lt : 0.f;
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) acc[nb] *= inv;
        }
        tile_store_sums<H, D>(t, piece[t.wv], acc, o, ws_acc);
    }
    if (g == 0 && t.member.x >= 0) {
        if (t.member.y < 0) {
            lse[(size_t)t.member.x * H + t.head] = has_sum<MOD>(lt) ? mref + log2f(lt) : 0.f;
        } else {
            ws_ml[((size_t)t.member.y * H + t.head) * 2] = mref;
            ws_ml[((size_t)t.member.y * H + t.head) * 2 + 1] = lt;
        }
    }
}

// Destination side.  PDS: (p, ds) of the pairs go to the scratch for the source side that reads them back; otherwise that side
// forms them again (k_attn_bwd_src_tile_bf16_again) and all it is handed is (lse, delta) of the rows, `stat` (n, H): the
// segments of a split row write the same values.
// MOD without a score term: delta = dO . O with O as stored is off by O's rounding and by that of the p that O was summed with, both 2^-9 of each
// term, which all pairs of a row share: at L = 32768, k = 8 dq and dk come out 0.0041 off (0.0017 is one rounding of the result) and the slopes'
// gradient, a sum over all pairs that nothing rounds, as far.  The pairs of a whole row give delta in 32 bits, sum p dP / sum p, once they have all been seen:
//   ds = p (dP - delta') du  corrected by  (delta' - delta) sum p du K  in dq and by  (delta' - delta) sum p |pos - pos|  in the slopes' gradient,
// the source side is handed delta.  (The sum of p, 1 but for the rounding of lse, keeps the sum of ds over a row at zero, by which distances in the hundreds multiply.)
// With a score term the pairs leave for the source side as they are formed, so dq, dk and dv keep delta', the slopes' gradient does not (tile_slope_fix).
// One more product a block over the K rows at hand.  The segments of a split row leave their sums, that of p du K rounded to bfloat16 (2^-9 of a
// correction that is 2^-8 of dq): k_score_split forms delta and the slopes' correction before the source side runs, k_score_merge dq's.
template <int H, int D, int HW, int WPE, bool DROP, int BIAS, bool PDS, int SP, bool MOD = false>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(MOD ? WPE - 2 : DROP || BIAS ? WPE - 1 : WPE))) void k_attn_bwd_dst_rows_bf16(
    bpt_plan P, const bf16_t *__restrict__ q, const bf16_t *__restrict__ k, const bf16_t *__restrict__ v, const bf16_t *__restrict__ o,
    const bf16_t *__restrict__ d_o, const float *__restrict__ lse, bf16_t *__restrict__ dq, uint32_t *__restrict__ pds,
    float2 *__restrict__ stat, float *__restrict__ ws_dq, float scale, float scale_log2e, uint32_t drop_thr, uint32_t drop_seed, float drop_inv,
    const float *__restrict__ bias, float *__restrict__ ds_out, typename ModArg<MOD>::type md) {
    static_assert(PDS || BIAS == 0, "the score term's gradient is stored by the pair's position");
    constexpr uint32_t RB = H * D * 2;
    constexpr bool FIX = MOD && !PDS;                             // delta from the pairs (comment above)
    const Narrow nw{};
    TileCtx t;
    if (!tile_begin<bf16_t, H, D, HW, false, SP>(P, t, nw)) return;
    __shared__ int2 ent_lds[HW][TILE_CHUNK];
    __shared__ int fst_lds[HW][PDS ? TILE_CHUNK : 1];
    int2 *ent = ent_lds[t.wv];
    int *fst = PDS ? fst_lds[t.wv] : nullptr;
    constexpr int PIECE = 2 * TILE_ROWS_FLOATS_BF16 + 4 * TILE_R;      // (the turned sums' rows are longer)
    static_assert(PIECE >= TILE_PART_FLOATS && PIECE >= TILE_R * TILE_TURN_STRIDE, "parts and turned sums fit the rows' piece");
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    __shared__ __attribute__((aligned(16))) float pos_lds[HW][MOD ? TILE_R : 4];
    char *const k_lds = reinterpret_cast<char *>(piece[t.wv]), *const v_lds = k_lds + 4 * TILE_ROWS_FLOATS_BF16;
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const char *kb = reinterpret_cast<const char *>(k), *vb = reinterpret_cast<const char *>(v);
    uint32_t *const pds_h = pds + (size_t)t.head * (size_t)P.n_edges;     // this head's part of the scratch
    Bf8 qb[2], dob[2];
    float delta, lse_c;
    {
        uint32_t off[2];
        tile_member_offsets<RB>(t, off);
        uintx4v qr[2], dr[2], orow[2];
        tile_ask_rows_bf16(reinterpret_cast<const char *>(d_o), off, dr);
        tile_ask_rows_bf16(reinterpret_cast<const char *>(o), off, orow);
        tile_ask_rows_bf16(reinterpret_cast<const char *>(q), off, qr);
        const size_t at = (size_t)max(t.member.x, 0) * H + t.head;
        lse_c = g == 0 ? lse[at] : 0.f;
        float part[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            part[r] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                part[r] = fmaf(__uint_as_float(dr[r][i] << 16), __uint_as_float(orow[r][i] << 16), part[r]);
                part[r] = fmaf(__uint_as_float(dr[r][i] & 0xffff0000u), __uint_as_float(orow[r][i] & 0xffff0000u), part[r]);
            }
            part[r] = head_sum<8>(part[r]);                       // dO . O of member 8 r + l / 8, this head
        }
        tile_put_rows_bf16(k_lds, qr, t.lane);
        tile_put_rows_bf16(v_lds, dr, t.lane);
        wave_lds_fence();
        tile_operand_bf16(k_lds, c, g, qb);
        tile_operand_bf16(v_lds, c, g, dob);
        wave_lds_fence();
        const float d0 = lane_bcast(part[0], 8 * (c & 7)), d1 = lane_bcast(part[1], 8 * (c & 7));
        delta = c < 8 ? d0 : d1;
        if constexpr (!PDS && !FIX) {
            if (g == 0 && t.part == 0 && t.member.x >= 0) stat[at] = make_float2(lse_c, delta);
        }
        lse_c = lane_bcast(lse_c, c);
    }
    float slope = 0.f, pos_m = 0.f, slope_sum = 0.f;
    if constexpr (MOD) {
        if (md.slopes) {
            slope = md.slopes[t.head] * LOG2E;
            pos_m = md.pos_member[max(t.member.x, 0)];
        }
    }
    floatx4v acc[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
    float dp_sum = 0.f, far_sum = 0.f, p_sum = 0.f;
    floatx4v pk[FIX ? 4 : 1];                                     // sum of p du K, laid out as acc
#pragma unroll
    for (int nb = 0; nb < (FIX ? 4 : 1); ++nb) pk[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
    struct Blk {
        uintx4v kr[2], vr[2];
        int xe[DROP || BIAS == 1 ? 4 : 1];
        float bz[BIAS ? 4 : 1];
        float pos;                                                // of entry c, in the first lane group
    };
    auto walk = [&](auto again) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(again)::value;
    if constexpr (CAREFUL) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        if (p0 != t.p_begin) tile_ask_entries(P, p0, cnt, t.lane, er);
        tile_put_entries(er, ent, cnt, t.lane, fst);
        auto numbers = [&](int b, const int (&mk)[4], uint32_t (&pos)[4]) {
            const int4 f4 = *reinterpret_cast<const int4 *>(&fst[TILE_R * b + 4 * g]);
            pos[0] = tile_pair_number(f4.x, mk[0], c); pos[1] = tile_pair_number(f4.y, mk[1], c);
            pos[2] = tile_pair_number(f4.z, mk[2], c); pos[3] = tile_pair_number(f4.w, mk[3], c);
        };
        auto issue = [&](Blk &B, int b) {
            if constexpr (DROP || BIAS == 1) tile_pair_eids(P, p0 + TILE_R * b + 4 * g, t.p_end, c, B.xe);
            if constexpr (MOD) {
                if (md.slopes && g == 0) B.pos = md.pos_entry[ent[TILE_R * b + c].x];
            }
            uint32_t off[2];
            tile_entry_offsets<RB>(t, ent + TILE_R * b, off);
            tile_ask_rows_bf16(kb, off, B.kr);
            tile_ask_rows_bf16(vb, off, B.vr);
            if constexpr (BIAS) {
                int mk[4];
                uint32_t pos[4];
                tile_masks(ent + TILE_R * b, g, mk);
                numbers(b, mk, pos);
#pragma unroll
                for (int r = 0; r < 4; ++r) B.bz[r] = bias[tile_bias_at<H, BIAS>(P, t.head, B.xe[BIAS == 1 ? r : 0], pos[r])];
            }
        };
        Blk B;
        issue(B, 0);
        for (int b = 0; b < nblk; ++b) {
            int mk[4], xe[DROP || BIAS == 1 ? 4 : 1];
            float bz[BIAS ? 4 : 1];
            uint32_t pos[4];
            tile_masks(ent + TILE_R * b, g, mk);
            if constexpr (PDS) numbers(b, mk, pos);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (DROP || BIAS == 1) xe[DROP || BIAS == 1 ? r : 0] = B.xe[DROP || BIAS == 1 ? r : 0];
                if constexpr (BIAS) bz[BIAS ? r : 0] = B.bz[BIAS ? r : 0];
            }
            tile_put_rows_bf16(k_lds, B.kr, t.lane);
            tile_put_rows_bf16(v_lds, B.vr, t.lane);
            if constexpr (MOD) {
                if (md.slopes && g == 0) pos_lds[t.wv][c] = B.pos;
            }
            wave_lds_fence();
            if (b + 1 < nblk) issue(B, b + 1);
            issue_loads_first();
            Bf8 row[2];
            tile_operand_bf16(k_lds, c, g, row);
            const floatx4v st = tile_dot_bf16(row, qb);
            tile_operand_bf16(v_lds, c, g, row);
            const floatx4v dp = tile_dot_bf16(row, dob);
            float ds[4], sm[4], du[4], pos_e[4], pdu[4];
            if constexpr (MOD) {
                float x[4];
                const floatx4v at_e = *reinterpret_cast<const floatx4v *>(&pos_lds[t.wv][4 * g]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = BIAS ? st[r] + bz[BIAS ? r : 0] : st[r];
                    pos_e[r] = at_e[r];
                }
                tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, sm, du);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float pe = where_pair_or_zero(mk[r], c, __builtin_amdgcn_exp2f(MOD ? sm[r] - lse_c : (BIAS ? st[r] + bz[BIAS ? r : 0] : st[r]) * scale_log2e - lse_c));
                float mt = 1.f;                                   // dropout multiplier of this pair (as in the forward)
                if constexpr (DROP)
                    mt = dropout_keep((uint32_t)xe[DROP ? r : 0] * (uint32_t)H + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
                if constexpr (MOD) {
                    const float x = where_pair_or_zero(mk[r], c, pe * (dp[r] * mt));
                    ds[r] = fmaf(-pe, delta, x);
                    if (md.part) {
                        const float far = fabsf(pos_m - pos_e[r]);
                        slope_sum += pair_if<CAREFUL>(mk[r], c, ds[r] * far);
                        far_sum += pair_if<CAREFUL>(mk[r], c, pe * far);
                        if constexpr (!FIX) {
                            dp_sum += pair_if<CAREFUL>(mk[r], c, ds[r]);
                            p_sum += pe;
                        }
                    }
                    ds[r] = pair_if<CAREFUL>(mk[r], c, ds[r] * du[r]);
                    if constexpr (FIX) {
                        dp_sum += x;
                        p_sum += pe;
                        pdu[r] = pair_if<CAREFUL>(mk[r], c, pe * du[r]);
                    }
                } else {
                    ds[r] = pe * (dp[r] * mt - delta) * scale;
                }
                pe *= mt;                                         // what multiplies v (forward) and dO (dV)
                if (PDS && ((mk[r] >> c) & 1)) {
                    pds_h[pos[r]] = pack_bf16(pe, ds[r]);
                    if constexpr (BIAS) ds_out[tile_bias_at<H, BIAS>(P, t.head, xe[BIAS == 1 ? r : 0], pos[r])] = ds[r];   // dL/d(score before scaling)
                }
            }
            if constexpr (CAREFUL) {
                tile_axpy_pairs_bf16(ds, mk, k_lds, c, g, acc);
                if constexpr (FIX) tile_axpy_pairs_bf16(pdu, mk, k_lds, c, g, pk);
            } else {
                Bf4 da;
                da.u[0] = pack_bf16(ds[0], ds[1]);
                da.u[1] = pack_bf16(ds[2], ds[3]);
                tile_axpy_rows_bf16(da, k_lds, c, g, acc);
                if constexpr (FIX) {
                    da.u[0] = pack_bf16(pdu[0], pdu[1]);
                    da.u[1] = pack_bf16(pdu[2], pdu[3]);
                    tile_axpy_rows_bf16(da, k_lds, c, g, pk);
                }
            }
            wave_lds_fence();                                     // (read before the next block's are written)
            issue_loads_first();
        }
    }
    };
    walk(std::false_type{});
    if constexpr (MOD) {
        if (tile_any_odd(tile_odd(acc) + tile_odd(pk) + (slope_sum + far_sum) * 0.f)) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int nb = 0; nb < (FIX ? 4 : 1); ++nb) pk[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
            slope_sum = far_sum = dp_sum = p_sum = 0.f;
            walk(std::true_type{});
        }
    }
    if constexpr (FIX) {
        float4 sums = make_float4(groups_sum(dp_sum), groups_sum(far_sum), groups_sum(p_sum), 0.f);      // of member c, of this part
        if constexpr (SP > 1) {
            __shared__ float4 meet[HW][TILE_R];
            tile_parts_sum<SP, HW>(meet, t, sums);
        }
        const bool segment = t.member.y >= 0;
        const float better = segment || sums.z == 0.f ? delta : sums.x / sums.z, less = delta == delta ? delta - better : 0.f;      // (NaN: the pairs, if there are any, are NaN as they are)
        slope_sum = fmaf(less, far_sum, slope_sum);
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) acc[nb] += less * pk[nb];
        if (g == 0 && t.part == 0 && t.member.x >= 0) {
            stat[(size_t)t.member.x * H + t.head] = make_float2(lse_c, better);
            if (segment) md.split[(size_t)t.member.y * H + t.head] = sums;
        }
        if (__builtin_amdgcn_ballot_w64(segment) != 0) {          // (the parts of a tile have the same members)
            tile_sums_by_row(piece[t.wv], pk, c, g);
            tile_put_low<SP, H, D, false>(md, t, piece[t.wv], piece[t.wv % (HW / SP)], (HW / SP) * PIECE, pk, nw);
        }
    }
    if constexpr (MOD) {
        if constexpr (!FIX) {
            if (md.part) tile_slope_fix<SP, HW>(md, t, H, dp_sum, far_sum, p_sum, slope_sum);
        }
        tile_put_slope_part<SP>(md, t, H, slope_sum);
    }
    if constexpr (SP > 1) {
        tile_sums_by_row(piece[t.wv], acc, c, g);
        tile_park(piece[t.wv], acc, t.lane);
        __syncthreads();
        tile_meet_and_store<SP, H, D, false>(piece[t.wv % (HW / SP)], (HW / SP) * PIECE, t, dq, ws_dq, nw);
    } else {
        tile_store_sums<H, D>(t, piece[t.wv], acc, dq, ws_dq);
    }
}

// Heads of fewer than 64 columns (their rows on 4 bytes): rows of 8 bytes a lane, kept in registers.
template <int H, int D, int HW, int WPE, bool DROP, int SP, bool MOD = false>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(MOD ? WPE - 1 : WPE))) void k_attn_fwd_tile_bf16(
    bpt_plan P, const bf16_t *__restrict__ q, const bf16_t *__restrict__ k, const bf16_t *__restrict__ v, bf16_t *__restrict__ o,
    float *__restrict__ lse, float *__restrict__ ws_acc, float *__restrict__ ws_ml, float scale_log2e, uint32_t drop_thr,
    uint32_t drop_seed, float drop_inv, Narrow nw, Keep keep, typename ModArg<MOD>::type md) {
    const int Hs = nw.h;                                          // heads as lse, workspace and dropout keys count them
    const uint32_t RB = (uint32_t)(nw.heads * nw.d) * 2;          // bytes of a node row
    const int block = keep_or_tile<HW * WAVE>(keep);
    if (block < 0) return;
    bf16_t *const o_keep = reinterpret_cast<bf16_t *>(keep.o);
    TileCtx t;
    if (!tile_begin<bf16_t, H, D, HW, true, SP>(P, t, nw, (unsigned)block)) return;
    __shared__ int2 ent_lds[HW][TILE_CHUNK];
    int2 *ent = ent_lds[t.wv];
    constexpr int PIECE = SP > 1 ? TILE_PART_FWD_FLOATS : TILE_KT_FLOATS_BF16;
    static_assert(PIECE >= TILE_KT_FLOATS_BF16, "the rows fit");
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    __shared__ __attribute__((aligned(16))) float pos_lds[HW][MOD ? TILE_R : 4];      // positions of the block's entries
    char *kt = reinterpret_cast<char *>(piece[t.wv]);
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const uint32_t offr = t.offa, offc = t.offv;
    const char *kb = reinterpret_cast<const char *>(k), *vb = reinterpret_cast<const char *>(v);
    Bf8 qb[2];
    tile_load_row_bf16(reinterpret_cast<const char *>(q) + (size_t)max(t.member.x, 0) * RB + offr, qb, g, nw);
    float slope = 0.f, pos_m = 0.f;
    if constexpr (MOD) {
        if (md.slopes) {
            slope = md.slopes[t.head] * LOG2E;
            pos_m = md.pos_member[max(t.member.x, 0)];
        }
    }
    floatx4v acc[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
    float mref = m_init<MOD>(), lrun = 0.f;
    bool fresh = true;                                            // nothing has been summed up yet
    struct Blk {
        uint2 kq[4];                                              // columns 4 c .. 4 c + 3 of the K rows of entries 4 g + r
        uint2 vr[4];
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
        auto issue_k = [&](Blk &B, int b) {
            const int4 e01 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g]);
            const int4 e23 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g + 2]);
            const int idxv[4] = {e01.x, e01.z, e23.x, e23.z};
#pragma unroll
            for (int r = 0; r < 4; ++r) B.kq[r] = tile_row4_bf16<true>(kb + ((uint32_t)idxv[r] * RB + offc));
        };
        auto issue_rest = [&](Blk &B, int b) {
            if constexpr (MOD) {
                if (md.slopes && g == 0) B.pos = md.pos_entry[ent[TILE_R * b + c].x];
            }
            if constexpr (DROP) tile_pair_eids(P, p0 + TILE_R * b + 4 * g, t.p_end, c, B.xe);
            const int4 e01 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g]);
            const int4 e23 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g + 2]);
            const int idxv[4] = {e01.x, e01.z, e23.x, e23.z};
            B.mk[0] = e01.y; B.mk[1] = e01.w; B.mk[2] = e23.y; B.mk[3] = e23.w;
#pragma unroll
            for (int r = 0; r < 4; ++r) B.vr[r] = tile_row4_bf16<true>(vb + ((uint32_t)idxv[r] * RB + offc));
        };
        auto compute = [&](const Blk &B) {
            Bf8 kr[2];
            if constexpr (MOD) {
                if (md.slopes && g == 0) pos_lds[t.wv][c] = B.pos;
            }
            tile_rows_to_operand_bf16(kt, B.kq, c, g, kr, nw);
            const floatx4v st = tile_dot_bf16(kr, qb);
            float sc[4];
            if constexpr (MOD) {
                const floatx4v at_e = *reinterpret_cast<const floatx4v *>(&pos_lds[t.wv][4 * g]);
                const float pos_e[4] = {at_e[0], at_e[1], at_e[2], at_e[3]}, x[4] = {st[0], st[1], st[2], st[3]};
                float du[4];
                tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, sc, du);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[r] = where_pair(B.mk[r], c, sc[r]);
            } else
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[r] = where_pair(B.mk[r], c, st[r] * scale_log2e);
            const float mb = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
            if (__builtin_amdgcn_ballot_w64(mb > mref + MFMA_TAU) != 0) {
                const float mn = fmaxf(mref, groups_max(mb));    // over the four lanes of member c
                const float al = __builtin_amdgcn_exp2f(mref - mn);
                mref = mn;
                if (!fresh) {
                    lrun *= al;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float a = lane_bcast(al, 4 * g + r);
#pragma unroll
                        for (int nb = 0; nb < 4; ++nb) acc[nb][r] *= a;
                    }
                }
            }
            fresh = false;
            float pr[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pr[r] = __builtin_amdgcn_exp2f(sc[r] - mref);
                lrun += pr[r];                                   // the softmax denominator ignores dropout
                if constexpr (DROP)
                    pr[r] *= dropout_keep((uint32_t)B.xe[DROP ? r : 0] * (uint32_t)Hs + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
            }
            if constexpr (CAREFUL) {
                tile_axpy_pairs(pr, B.mk, B.vr, c, g, acc);
            } else {
                Bf4 pa;
                pa.u[0] = pack_bf16(pr[0], pr[1]);
                pa.u[1] = pack_bf16(pr[2], pr[3]);
                tile_axpy_bf16(pa, B.vr, acc);
            }
        };
        auto issue = [&](Blk &B, int b) { issue_k(B, b); issue_rest(B, b); };
        if constexpr (DROP) tile_walk<Blk>(nblk, issue, compute);      // (the K rows ahead: eight registers more)
        else tile_walk_first_ahead<Blk>(nblk, issue_k, issue_rest, compute, []() {});
        wave_lds_fence();
    }
    };
    walk(std::false_type{});
    if constexpr (MOD) {
        if (tile_any_odd(tile_odd(acc))) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
            mref = m_init<MOD>();
            lrun = 0.f;
            fresh = true;
            walk(std::true_type{});
        }
    }
    float lt = groups_sum(lrun);
    if constexpr (SP > 1) {
        tile_meet_forward<SP, H, D, true, MOD>(piece[t.wv], piece[t.wv % (HW / SP)], (HW / SP) * PIECE, t, acc, mref, lt, o, ws_acc, nw, o_keep);
        if (t.part != 0) return;
    } else {
        tile_store_rows<H, D, true, true>(t, acc, has_sum<MOD>(lt) ? 1.f / lt : 0.f, o, ws_acc, nw, o_keep);
    }
    if (g == 0 && t.member.x >= 0) {
        if (t.member.y < 0) {
            lse[(size_t)t.member.x * Hs + t.head] = has_sum<MOD>(lt) ? mref + log2f(lt) : 0.f;
        } else {
            ws_ml[((size_t)t.member.y * Hs + t.head) * 2] = mref;
            ws_ml[((size_t)t.member.y * Hs + t.head) * 2 + 1] = lt;
        }
    }
}

// Destination side of such heads: (p, ds) of the pairs go to the scratch.
template <int H, int D, int HW, int WPE, bool DROP, int SP>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(DROP ? WPE - 1 : WPE))) void k_attn_bwd_dst_tile_bf16(
    bpt_plan P, const bf16_t *__restrict__ q, const bf16_t *__restrict__ k, const bf16_t *__restrict__ v, const bf16_t *__restrict__ o,
    const bf16_t *__restrict__ d_o, const float *__restrict__ lse, bf16_t *__restrict__ dq, uint32_t *__restrict__ pds,
    float *__restrict__ ws_dq, float scale, float scale_log2e, uint32_t drop_thr, uint32_t drop_seed, float drop_inv, Narrow nw) {
    const int Hs = nw.h;
    const uint32_t RB = (uint32_t)(nw.heads * nw.d) * 2;
    TileCtx t;
    if (!tile_begin<bf16_t, H, D, HW, true, SP>(P, t, nw)) return;
    __shared__ int2 ent_lds[HW][TILE_CHUNK];
    __shared__ int fst_lds[HW][TILE_CHUNK];
    int2 *ent = ent_lds[t.wv];
    int *fst = fst_lds[t.wv];
    constexpr int PIECE = SP > 1 ? TILE_PART_FLOATS : TILE_KT_FLOATS_BF16;
    static_assert(PIECE >= TILE_KT_FLOATS_BF16, "the rows fit");
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    char *kt = reinterpret_cast<char *>(piece[t.wv]);
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const uint32_t offr = t.offa, offc = t.offv;
    const char *kb = reinterpret_cast<const char *>(k), *vb = reinterpret_cast<const char *>(v);
    const size_t mrow = (size_t)max(t.member.x, 0) * RB + offr;
    uint32_t *const pds_h = pds + (size_t)t.head * (size_t)P.n_edges;     // this head's part of the scratch
    Bf8 qb[2], dob[2];
    float delta, lse_c;
    {
        Bf8 ob[2];
        tile_load_row_bf16(reinterpret_cast<const char *>(q) + mrow, qb, g, nw);
        tile_load_row_bf16(reinterpret_cast<const char *>(d_o) + mrow, dob, g, nw);
        tile_load_row_bf16(reinterpret_cast<const char *>(o) + mrow, ob, g, nw);
        float part = 0.f;
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
            const uint32_t a[4] = {dob[h2].q.x, dob[h2].q.y, dob[h2].q.z, dob[h2].q.w}, b[4] = {ob[h2].q.x, ob[h2].q.y, ob[h2].q.z, ob[h2].q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                part = fmaf(__uint_as_float(a[i] << 16), __uint_as_float(b[i] << 16), part);
                part = fmaf(__uint_as_float(a[i] & 0xffff0000u), __uint_as_float(b[i] & 0xffff0000u), part);
            }
        }
        delta = groups_sum(part);                                 // dO . O of member c, this head
        lse_c = lse[(size_t)max(t.member.x, 0) * Hs + t.head];
    }
    floatx4v acc[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) acc[nb] = floatx4v{0.f, 0.f, 0.f, 0.f};
    struct Blk {
        uint2 kc[4], vc[4];                                       // columns 4 c .. 4 c + 3 of the K / V rows of entries 4 g + r
        int mk[4];                                                // bit c of mk[r]: the pair (entry 4 g + r, member c) exists
        uint32_t pos[4];
        int xe[DROP ? 4 : 1];
    };
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        if (p0 != t.p_begin) tile_ask_entries(P, p0, cnt, t.lane, er);
        tile_put_entries(er, ent, cnt, t.lane, fst);
        auto issue = [&](Blk &B, int b) {
            if constexpr (DROP) tile_pair_eids(P, p0 + TILE_R * b + 4 * g, t.p_end, c, B.xe);
            const int4 e01 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g]);
            const int4 e23 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g + 2]);
            const int idxv[4] = {e01.x, e01.z, e23.x, e23.z};
            B.mk[0] = e01.y; B.mk[1] = e01.w; B.mk[2] = e23.y; B.mk[3] = e23.w;
            const int4 f4 = *reinterpret_cast<const int4 *>(&fst[TILE_R * b + 4 * g]);
            B.pos[0] = tile_pair_number(f4.x, e01.y, c); B.pos[1] = tile_pair_number(f4.y, e01.w, c);
            B.pos[2] = tile_pair_number(f4.z, e23.y, c); B.pos[3] = tile_pair_number(f4.w, e23.w, c);
#pragma unroll
            for (int r = 0; r < 4; ++r) B.kc[r] = tile_row4_bf16<true>(kb + ((uint32_t)idxv[r] * RB + offc));
#pragma unroll
            for (int r = 0; r < 4; ++r) B.vc[r] = tile_row4_bf16<true>(vb + ((uint32_t)idxv[r] * RB + offc));
        };
        auto compute = [&](const Blk &B) {
            Bf8 kr[2];
            tile_rows_to_operand_bf16(kt, B.kc, c, g, kr, nw);
            const floatx4v st = tile_dot_bf16(kr, qb);
            tile_rows_to_operand_bf16(kt, B.vc, c, g, kr, nw);
            const floatx4v dp = tile_dot_bf16(kr, dob);
            float ds[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float pe = where_pair_or_zero(B.mk[r], c, __builtin_amdgcn_exp2f(st[r] * scale_log2e - lse_c));
                float mt = 1.f;                                   // dropout multiplier of this pair (as in the forward)
                if constexpr (DROP)
                    mt = dropout_keep((uint32_t)B.xe[DROP ? r : 0] * (uint32_t)Hs + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
                ds[r] = pe * (dp[r] * mt - delta) * scale;
                pe *= mt;                                         // what multiplies v (forward) and dO (dV)
                if ((B.mk[r] >> c) & 1) pds_h[B.pos[r]] = pack_bf16(pe, ds[r]);
            }
            Bf4 da;
            da.u[0] = pack_bf16(ds[0], ds[1]);
            da.u[1] = pack_bf16(ds[2], ds[3]);
            tile_axpy_bf16(da, B.kc, acc);
        };
        tile_walk<Blk>(nblk, issue, compute);
        wave_lds_fence();
    }
    if constexpr (SP > 1) {
        tile_park(piece[t.wv], acc, t.lane);
        __syncthreads();
        tile_meet_and_store<SP, H, D, true>(piece[t.wv % (HW / SP)], (HW / SP) * PIECE, t, dq, ws_dq, nw);
    } else {
        tile_store_rows<H, D, false, true>(t, acc, 1.f, dq, ws_dq, nw);
    }
}

constexpr int TILE_WT_STRIDE_BF16 = 20;
template <int H, int D, int HW, int WPE, bool NARROW = false, int SP = 1, bool MOD = false>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(WPE))) void k_attn_bwd_src_tile_bf16(
    bpt_plan P, const bf16_t *__restrict__ q, const bf16_t *__restrict__ d_o, const uint32_t *__restrict__ pds, bf16_t *__restrict__ dk,
    bf16_t *__restrict__ dv, float *__restrict__ ws_dk, float *__restrict__ ws_dv, Narrow nw) {
    const uint32_t RB = NARROW ? (uint32_t)(nw.heads * nw.d) * 2 : (uint32_t)(H * D * 2);
    TileCtx t;
    if (!tile_begin<bf16_t, H, D, HW, NARROW, SP>(P, t, nw)) return;
    constexpr int ENT = TILE_CHUNK * 2, LIVE = ENT + TILE_R * TILE_WT_STRIDE_BF16, PIECE = SP > 1 ? 2 * TILE_PART_FLOATS : LIVE;
    static_assert(PIECE >= LIVE, "the lists fit");
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    int2 *ent = reinterpret_cast<int2 *>(piece[t.wv]);
    uint32_t *const wt = reinterpret_cast<uint32_t *>(piece[t.wv] + ENT);         // (turned as in the float32 kernel)
    const int c = t.c, g = t.g;
    const uint32_t offc = t.offv;
    const char *qb = reinterpret_cast<const char *>(q), *db = reinterpret_cast<const char *>(d_o);
    const uint32_t *const pds_h = pds + (size_t)t.head * (size_t)P.n_edges;
    floatx4v ak[4], av[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) { ak[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; av[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
    struct Blk {
        uint2 qr[4], dr[4];
        uint32_t w[4];                                            // (p, ds) of the pairs (entry c, member 4 g + r)
        int mk[4];                                                // bit c of mk[r]: the pair (entry 4 g + r, member c) exists
    };
    auto walk = [&](auto again) __attribute__((always_inline)) {
    constexpr bool CAREFUL = decltype(again)::value;
    for (int p0 = t.p_begin; p0 < t.p_end; p0 += TILE_CHUNK) {
        const int cnt = min(TILE_CHUNK, t.p_end - p0), nblk = (cnt + TILE_R - 1) / TILE_R;
        tile_stage_entries(P, ent, p0, cnt, t.lane);
        // (the positions of a block's pairs in the scratch are fetched one block ahead, as in the float32 kernel, so that the
        // (p, ds) loads leave with the row loads; positions past the group's end are read at its last entry: their masks are
        // empty.  The four registers this takes are why the kernel is compiled for five wavefronts per SIMD, not six: with
        // six it spills and loses what the prefetch gains)
        auto positions = [&](int b, int (&pos)[4]) { tile_pair_positions(P, min(p0 + TILE_R * b + c, t.p_end - 1), g, pos); };
        int pos_ahead[4], ahead_of = -1;
        auto issue = [&](Blk &B, int b) {
            const int4 e01 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g]);
            const int4 e23 = *reinterpret_cast<const int4 *>(&ent[TILE_R * b + 4 * g + 2]);
            const int idxv[4] = {e01.x, e01.z, e23.x, e23.z};
            B.mk[0] = e01.y; B.mk[1] = e01.w; B.mk[2] = e23.y; B.mk[3] = e23.w;
            int pos[4];
            if (b == ahead_of) {
#pragma unroll
                for (int r = 0; r < 4; ++r) pos[r] = pos_ahead[r];
            } else {
                positions(b, pos);
            }
            if (b + 1 < nblk) positions(b + 1, pos_ahead);
            ahead_of = b + 1;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t off = (uint32_t)idxv[r] * RB + offc;
                B.qr[r] = tile_row4_bf16<NARROW>(qb + off);
                B.dr[r] = tile_row4_bf16<NARROW>(db + off);
                B.w[r] = pds_h[(uint32_t)pos[r]];
            }
        };
        auto compute = [&](const Blk &B) {
            *reinterpret_cast<uintx4v *>(wt + c * TILE_WT_STRIDE_BF16 + 4 * g) = uintx4v{B.w[0], B.w[1], B.w[2], B.w[3]};
            wave_lds_fence();
            uint32_t w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = wt[(4 * g + r) * TILE_WT_STRIDE_BF16 + c];
            wave_lds_fence();                                     // (read before the next block's are written)
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] &= (uint32_t)__builtin_amdgcn_sbfe(B.mk[r], c, 1);       // the scratch of pairs that do not exist is not initialised
            if constexpr (CAREFUL) {
                float pe[4], ds[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) { pe[r] = __uint_as_float(w[r] << 16); ds[r] = __uint_as_float(w[r] & 0xffff0000u); }
                tile_axpy_pairs(ds, B.mk, B.qr, c, g, ak);
                tile_axpy_pairs(pe, B.mk, B.dr, c, g, av);
            } else {
                Bf4 pa, da;
                pa.u[0] = pack_lo16(w[0], w[1]); pa.u[1] = pack_lo16(w[2], w[3]);
                da.u[0] = pack_hi16(w[0], w[1]); da.u[1] = pack_hi16(w[2], w[3]);
                tile_axpy_bf16(da, B.qr, ak);
                tile_axpy_bf16(pa, B.dr, av);
            }
        };
        tile_walk<Blk>(nblk, issue, compute);
        wave_lds_fence();
    }
    };
    walk(std::false_type{});
    if constexpr (MOD) {
        if (tile_any_odd(tile_odd(ak) + tile_odd(av))) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) { ak[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; av[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
            walk(std::true_type{});
        }
    }
    if constexpr (SP > 1) {
        constexpr int NEXT = (HW / SP) * PIECE;
        tile_park(piece[t.wv], ak, t.lane);
        tile_park(piece[t.wv] + TILE_PART_FLOATS, av, t.lane);
        __syncthreads();
        const float *const part0 = piece[t.wv % (HW / SP)];
        tile_meet_and_store<SP, H, D, NARROW>(part0, NEXT, t, dk, ws_dk, nw);
        tile_meet_and_store<SP, H, D, NARROW>(part0 + TILE_PART_FLOATS, NEXT, t, dv, ws_dv, nw);
    } else {
        tile_store_rows<H, D, false, NARROW>(t, ak, 1.f, dk, ws_dk, nw);
        tile_store_rows<H, D, false, NARROW>(t, av, 1.f, dv, ws_dv, nw);
    }
}

// Source side without the scratch: p and ds of a block's pairs are formed again from the entries' q and dO rows, which are
// loaded for the products over the entries anyway and turned in LDS, the members' k and v rows (held as operands) and the
// entries' (lse, delta), which the destination side leaves in `stat` (n, H).
// Why: the scratch holds 4 bytes per pair and head, as much as the node tensors on a dense graph, and reading it back is a
// gather of 4-byte words over 16 to 32 cache lines per instruction.  At L = 32768, k = 8, 16 heads the stores cost the
// destination side 70 of 295 us and the gathers this side 105 of 370 (the kernels without them, timing only); four more
// bfloat16 matrix instructions and two turns in LDS per block cost 70: 295 + 370 -> 237 + 315 us, the step 890 -> 782.
// Both backward kernels together at 8 heads: L = 8192, k = 4 60.8 -> 57.0 us; L = 4096, k = 32 64.7 -> 48.7; window 128 39.7 ->
// 30.9; L = 32768, k = 2 235 -> 221; 32-graph batch 102.5 -> 99.2; L = 512 and L = 8192 with dropout level.  (6 heads of 50
// columns with dropout lost 2 %: heads of fewer than 64 columns keep the scratch.)  float32 keeps it too: there the two
// products are 1024 cycles of the matrix pipeline per block.  122 registers: compiled for four wavefronts per SIMD.
template <int H, int D, int HW, int WPE, bool DROP, int SP = 1, bool MOD = false>
__global__ __launch_bounds__(HW * WAVE) __attribute__((amdgpu_waves_per_eu(MOD ? WPE - 1 : WPE))) void k_attn_bwd_src_tile_bf16_again(
    bpt_plan P, const bf16_t *__restrict__ q, const bf16_t *__restrict__ k, const bf16_t *__restrict__ v, const bf16_t *__restrict__ d_o,
    const float2 *__restrict__ stat, bf16_t *__restrict__ dk, bf16_t *__restrict__ dv, float *__restrict__ ws_dk, float *__restrict__ ws_dv,
    float scale, float scale_log2e, uint32_t drop_thr, uint32_t drop_seed, float drop_inv, typename ModArg<MOD>::type md) {
    constexpr uint32_t RB = H * D * 2;
    const Narrow nw{};
    TileCtx t;
    if (!tile_begin<bf16_t, H, D, HW, false, SP>(P, t, nw)) return;
    // a wavefront's piece: its entry list, the rows being turned, the entries' (lse, delta); afterwards (SP > 1) what it has summed up
    constexpr int ENT = TILE_CHUNK * 2, ROWS = 2 * TILE_ROWS_FLOATS_BF16 + 4 * TILE_R, LIVE = ENT + ROWS + 2 * TILE_R, PIECE = SP > 1 ? 2 * TILE_PART_FLOATS : LIVE;
    static_assert(PIECE >= LIVE && ROWS >= TILE_R * TILE_TURN_STRIDE, "the lists and the turned sums fit");
    __shared__ __attribute__((aligned(16))) float piece[HW][PIECE];
    __shared__ __attribute__((aligned(16))) float pos_lds[HW][MOD ? TILE_R : 4];
    int2 *ent = reinterpret_cast<int2 *>(piece[t.wv]);
    char *const q_lds = reinterpret_cast<char *>(piece[t.wv] + ENT), *const d_lds = q_lds + 4 * TILE_ROWS_FLOATS_BF16;
    float2 *const st_lds = reinterpret_cast<float2 *>(piece[t.wv] + ENT + ROWS);
    TileEntryRegs er;
    if (t.p_end > t.p_begin) tile_ask_entries(P, t.p_begin, min(TILE_CHUNK, t.p_end - t.p_begin), t.lane, er);
    issue_loads_first();
    const int c = t.c, g = t.g;
    const char *qb = reinterpret_cast<const char *>(q), *db = reinterpret_cast<const char *>(d_o);
    const float2 *const stat_h = stat + t.head;
    Bf8 kb[2], vb[2];
    {
        uint32_t off[2];
        uintx4v kr[2], vr[2];
        tile_member_offsets<RB>(t, off);
        tile_ask_rows_bf16(reinterpret_cast<const char *>(k), off, kr);
        tile_ask_rows_bf16(reinterpret_cast<const char *>(v), off, vr);
        tile_put_rows_bf16(q_lds, kr, t.lane);
        tile_put_rows_bf16(d_lds, vr, t.lane);
        wave_lds_fence();
        tile_operand_bf16(q_lds, c, g, kb);
        tile_operand_bf16(d_lds, c, g, vb);
        wave_lds_fence();
    }
    float slope = 0.f, pos_m = 0.f;
    if constexpr (MOD) {
        if (md.slopes) {
            slope = md.slopes[t.head] * LOG2E;
            pos_m = md.pos_member[max(t.member.x, 0)];
        }
    }
    floatx4v ak[4], av[4];
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) { ak[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; av[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
    struct Blk {
        uintx4v qr[2], dr[2];
        float2 ld;                                                // (lse, delta) of entry c, in the first lane group
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
            if constexpr (MOD) {
                if (md.slopes && g == 0) B.pos = md.pos_entry[ent[TILE_R * b + c].x];
            }
            if (g == 0) B.ld = stat_h[(size_t)ent[TILE_R * b + c].x * H];
            uint32_t off[2];
            tile_entry_offsets<RB>(t, ent + TILE_R * b, off);
            tile_ask_rows_bf16(qb, off, B.qr);
            tile_ask_rows_bf16(db, off, B.dr);
        };
        Blk B;
        issue(B, 0);
        for (int b = 0; b < nblk; ++b) {
            int mk[4], xe[DROP ? 4 : 1];
            tile_masks(ent + TILE_R * b, g, mk);
#pragma unroll
            for (int r = 0; r < (DROP ? 4 : 0); ++r) xe[r] = B.xe[r];
            tile_put_rows_bf16(q_lds, B.qr, t.lane);
            tile_put_rows_bf16(d_lds, B.dr, t.lane);
            if (g == 0) st_lds[c] = B.ld;
            if constexpr (MOD) {
                if (md.slopes && g == 0) pos_lds[t.wv][c] = B.pos;
            }
            wave_lds_fence();
            if (b + 1 < nblk) issue(B, b + 1);
            issue_loads_first();
            Bf8 row[2];
            tile_operand_bf16(q_lds, c, g, row);
            const floatx4v st = tile_dot_bf16(row, kb);
            const floatx4v l01 = *reinterpret_cast<const floatx4v *>(&st_lds[4 * g]), l23 = *reinterpret_cast<const floatx4v *>(&st_lds[4 * g + 2]);
            const float lse_e[4] = {l01[0], l01[2], l23[0], l23[2]}, delta_e[4] = {l01[1], l01[3], l23[1], l23[3]};
            tile_operand_bf16(d_lds, c, g, row);
            const floatx4v dp = tile_dot_bf16(row, vb);
            float pe[4], ds[4], sm[4], du[4];
            if constexpr (MOD) {
                const floatx4v at_e = *reinterpret_cast<const floatx4v *>(&pos_lds[t.wv][4 * g]);
                const float pos_e[4] = {at_e[0], at_e[1], at_e[2], at_e[3]}, x[4] = {st[0], st[1], st[2], st[3]};
                tile_mod_scores(md, scale_log2e, slope, pos_m, pos_e, x, sm, du);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float p = where_pair_or_zero(mk[r], c, __builtin_amdgcn_exp2f((MOD ? sm[r] : st[r] * scale_log2e) - lse_e[r]));
                float mt = 1.f;                                   // dropout multiplier of this pair (as in the forward)
                if constexpr (DROP)
                    mt = dropout_keep((uint32_t)xe[DROP ? r : 0] * (uint32_t)H + (uint32_t)t.head, drop_seed, drop_thr, drop_inv);
                ds[r] = where_pair_or_zero(mk[r], c, MOD ? p * (dp[r] * mt - delta_e[r]) * du[r] : p * (dp[r] * mt - delta_e[r]) * scale);
                pe[r] = p * mt;
            }
            if constexpr (CAREFUL) {
                tile_axpy_pairs_bf16(ds, mk, q_lds, c, g, ak);
                tile_axpy_pairs_bf16(pe, mk, d_lds, c, g, av);
            } else {
                Bf4 pa, da;
                da.u[0] = pack_bf16(ds[0], ds[1]); da.u[1] = pack_bf16(ds[2], ds[3]);
                pa.u[0] = pack_bf16(pe[0], pe[1]); pa.u[1] = pack_bf16(pe[2], pe[3]);
                tile_axpy_rows_bf16(da, q_lds, c, g, ak);
                tile_axpy_rows_bf16(pa, d_lds, c, g, av);
            }
            wave_lds_fence();                                     // (read before the next block's are written)
            issue_loads_first();
        }
    }
    };
    walk(std::false_type{});
    if constexpr (MOD) {
        if (tile_any_odd(tile_odd(ak) + tile_odd(av))) {      // (what does not exist must not reach the sums: tile_odd)
#pragma unroll
            for (int nb = 0; nb < 4; ++nb) { ak[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; av[nb] = floatx4v{0.f, 0.f, 0.f, 0.f}; }
            walk(std::true_type{});
        }
    }
    float *const turn = reinterpret_cast<float *>(q_lds);
    if constexpr (SP > 1) {
        tile_sums_by_row(turn, ak, c, g);
        tile_sums_by_row(turn, av, c, g);
        constexpr int NEXT = (HW / SP) * PIECE;
        tile_park(piece[t.wv], ak, t.lane);
        tile_park(piece[t.wv] + TILE_PART_FLOATS, av, t.lane);
        __syncthreads();
        const float *const part0 = piece[t.wv % (HW / SP)];
        tile_meet_and_store<SP, H, D, false>(part0, NEXT, t, dk, ws_dk, nw);
        tile_meet_and_store<SP, H, D, false>(part0 + TILE_PART_FLOATS, NEXT, t, dv, ws_dv, nw);
    } else {
        tile_store_sums<H, D>(t, turn, ak, dk, ws_dk);
        tile_store_sums<H, D>(t, turn, av, dv, ws_dv);
    }
}

// ------------------------------------------------------------------------------------------
// host side: plans and arguments
// ------------------------------------------------------------------------------------------
inline int grid_for(const bpt_plan *p) { return (int)((p->n_items + WAVES_PER_BLOCK - 1) / WAVES_PER_BLOCK); }

inline int check_plan(const bpt_plan *p, bool need_idx) {
    if (!p) return BPT_ERR_NULL;
    if (p->n_rows < 0 || p->n_edges < 0 || p->n_items < 0 || p->n_heavy < 0 || p->n_slots < 0) return BPT_ERR_SIZE;
    if (p->n_items > 0 && (!p->items || !p->rowptr)) return BPT_ERR_NULL;
    if (p->n_edges > 0 && (!p->eid || (need_idx && !p->idx))) return BPT_ERR_NULL;
    if (p->n_heavy > 0 && !p->heavy) return BPT_ERR_NULL;
    if (p->n_items < p->n_rows) return BPT_ERR_SIZE;     // every row owns at least one item
    if (p->n_groups < 0 || p->grp_R < 0 || p->grp_R > 32 || p->n_grp_entries < 0) return BPT_ERR_SIZE;
    if (p->n_groups > 0 && (!p->grp_members || !p->grp_ptr || !p->grp_chunks || (p->n_edges > 0 && !p->grp_entries))) return BPT_ERR_NULL;
    if (p->n_groups > 0 && (p->grp_max_chunk < 1 || p->grp_max_chunk > p->n_groups)) return BPT_ERR_SIZE;
    if (p->n_index_nodes < 0) return BPT_ERR_SIZE;
    return BPT_OK;
}

inline int check_shape(int h, int d, int dtype) {
    if (dtype != BPT_F32 && dtype != BPT_F64 && dtype != BPT_BF16) return BPT_ERR_DTYPE;
    if (h < 1 || d < 1 || (int64_t)h * d > (1 << 20)) return BPT_ERR_SHAPE;
    return BPT_OK;
}

inline size_t acc_size(int dtype) { return dtype == BPT_F64 ? 8 : 4; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int launch_status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? BPT_OK : (int)e;
}

inline int64_t round16(int64_t b) { return (b + 15) & ~(int64_t)15; }

// dropout of the fused path: threshold on the 32-bit hash (0 = off), seed, 1 / (1 - p)
struct Dropout {
    uint32_t thr, seed;
    float inv;
};
inline Dropout make_dropout(float p, uint64_t seed) {
    if (!(p > 0.f)) return Dropout{0u, 0u, 1.f};
    const double t = (double)p * 4294967296.0;
    return Dropout{(uint32_t)(t >= 4294967295.0 ? 4294967295.0 : (t < 1.0 ? 1.0 : t)), (uint32_t)(seed ^ (seed >> 32)), 1.f / (1.f - p)};
}

// The row-group kernels address node rows and the per-pair scratch with 32-bit byte offsets.
inline bool fits32(int64_t n, int64_t unit) { return n >= 0 && n <= (int64_t)0xffffffffu / unit; }

inline int group_grid(const bpt_plan *P) { return (int)(8 * P->grp_max_chunk); }

// groups of 16 rows for the dense-tile kernels (one wavefront per head: h * 64 threads per workgroup)
inline bool has_tiles(const bpt_plan *P, int h, int d, size_t elem) {
    return P->n_groups > 0 && P->grp_R == TILE_R && P->grp_members && P->grp_ptr && P->grp_entries && P->grp_chunks &&
           P->grp_max_chunk > 0 && 8 * P->grp_max_chunk >= P->n_groups && P->n_grp_entries >= 0 && d == 64 && h <= 16 && (elem == 4 || elem == 2) &&
           fits32(std::max(P->n_rows, P->n_index_nodes), (int64_t)h * d * (int64_t)elem);
}

// Over how many wavefronts (1, 2 or 4) of a workgroup the blocks of a tile are spread.  A launch has 1024 SIMDs to fill, and one
// that does not lasts as long as its longest chain of blocks: each part's chain is a half or a quarter as long.  What
// the parts cost is the tile's header, read by each of them, and the meeting in LDS, so with more wavefronts than fill the chip
// a part has to keep enough blocks.  float32, 8 heads, forward / destination side / source side, one part -> two -> four:
//   584 wavefronts of 4 to 9 blocks (L = 512)           10.3 / 13.8 / 16.4 -> 8.0 / 10.8 / 10.9 -> 8.0 / 9.6 / 8.6 us
//   1032 of 9 (window of 128, L = 2048)                 20.5 / 29.8 / 17.0 -> 15.7 / 21.3 / 13.7 -> 14.5 / 19.4 / 13.8
//   1448 of 3 (L = 1400, k = 4)                         11.9 / 16.3 / 11.3 -> 11.4 / 14.3 / 10.2 -> 12.8 / 16.6 / 11.7
//   2056 of 9 (window of 128, L = 4096)                 25.2 / 38.6 / 25.1 -> 20.8 / 30.7 / 21.3 -> 22.9 / 32.5 / 22.3
//   2096 of 3 (16 heads, L = 1024, k = 4)               12.8 / 19.2 / 13.9 -> 13.4 / 19.6 / 15.0 -> 14.8 / 20.6 / 14.8
//   2072 of 4 / 2168 of 5 (L = 2048, k = 8)             16.8 / 26.1 / 19.0 -> 14.4 / 21.4 / 18.2 -> 15.8 / 22.4 / 17.5
//   4112 of 9 (window of 128, L = 8192)                 33.3 / 56.6 / 48.4 -> 32.3 / 53.1 / 35.5 -> 37.0 / 58.3 / 38.6
//   4160 of 5 / 4448 of 8 (L = 4096, k = 4, both ways)  24.0 / 37.6 / 37.0 -> 24.4 / 39.4 / 35.3 -> 27.8 / 42.4 / 37.1
//   8080 of 16 / 8072 of 9 (window of 256, L = 8192)    91.0 / 142 / 93.8  -> 93.2 / 140 / 85.0  -> 101 / 149 / 88.6
//   8256 of 5 (window of 64, L = 16384)                 46.5 / 72.1 / 51.4 -> 49.6 / 72.2 / 50.1 -> 57.4 / 84.7 / 61.6
// bfloat16, whose blocks are shorter against their headers:
//   552 of 5 (L = 512)      5.4 / 6.5 / 9.6 -> 5.1 / 5.7 / 7.3 -> 5.1 / 5.9 / 6.6;    1048 of 3    5.3 / 6.3 / 6.8 -> 5.7 / 6.4 / 7.2 -> 6.4 / 7.4 / 8.6
//   1032 of 9               9.6 / 11.8 / 9.0 -> 7.7 / 8.8 / 9.5 -> 7.6 / 8.4 / 10.2;  2056 of 9   10.6 / 14.1 / 11.5 -> 10.4 / 12.8 / 12.2 -> 12.0 / 14.2 / 14.4
//   2072 of 4               8.2 / 10.0 / 10.4 -> 7.9 / 10.2 / 11.9 -> 9.3 / 12.7 / 14.2;  4112 of 9   15.0 / 18.4 / 19.0 -> 16.6 / 20.0 / 21.9 -> 19.3 / 23.5 / 27.0
//   (two parts cost the last launches that take them up to 5 %: 1048 of 3)
// The same line holds with dropout, the score term and narrow heads (one head a workgroup in parts, two otherwise); float32:
//   L = 512, dropout                10.9 / 13.6 / 15.6 -> 7.9 / 10.2 / 10.4  -> 7.8 / 10.3 / 9.1;   term and dropout 11.8 / 16.5 / 16.2 -> 8.6 / 12.3 / 10.5 -> 8.0 / 11.9 / 8.2
//   window 128, L = 4096, dropout   27.9 / 39.4 / 24.5 -> 22.3 / 35.6 / 20.9 -> 25.0 / 37.2 / 22.6; 6 x 50 with dropout 34.8 / 37.8 / 21.7 -> 26.6 / 28.0 / 20.8 -> 26.8 / 30.9 / 19.9
//   L = 4096, k = 32, dropout       39.5 / 56.2 / 48.2 -> 34.8 / 54.5 / 43.6 -> 40.1 / 61.7 / 46.8; term and dropout 43.0 / 64.8 / 49.2 -> 37.5 / 63.9 / 45.1 -> 42.0 / 72.0 / 48.6
//                                   6 x 50 with dropout 55.9 / 59.4 / 42.7 -> 33.5 / 44.1 / 34.5 -> 38.4 / 49.3 / 37.4
//   L = 8192, k = 4 (one part)      35.8 / 55.6 / 38.3 -> 38.9 / 62.7 / 40.6;  6 x 50 with dropout 44.3 / 46.2 / 36.2 -> 47.0 / 50.1 / 38.4
// bfloat16, dropout: L = 512 6.3 / 7.0 / 12.8 -> 5.5 / 5.9 / 10.7 -> 5.5 / 6.2 / 7.8; window 128, L = 4096 13.2 / 14.1 / 16.6 -> 11.7 / 12.6 / 16.7 -> 13.8 /
// 15.4 / 18.8; 6 x 50 there 19.2 / 21.3 / 13.0 -> 14.4 / 17.3 / 12.8 -> 15.3 / 18.9 / 12.6.  Of 290 kernels of a hundred graphs drawn at random over all
// of these the rule slowed one by more than 1 % against one part (a window of 52, forward 16.9 -> 17.8).
// Two parts of launches that fill the chip about twice (6500 to 8192 wavefronts) pay on the source side (window 256, above) and with dropout
// (forward there 108.2 -> 106.8), not for a float32 forward without: L = 7000, k = 32 51.7 -> 53.9, L = 6000, k = 64 63.5 -> 66.0, window 128, L =
// 16000 61.1 -> 63.1, window 256 90.8 -> 92.4 (plain_forward; below, 5600 to 6300 wavefronts 42.7 -> 42.9, 46.2 -> 45.7, 48.4 -> 47.0).
inline int tile_parts(const bpt_plan *P, int heads, size_t elem, bool plain_forward = false) {
    const int64_t wavefronts = P->n_groups * heads, blocks = P->n_grp_entries / TILE_R;
    const int64_t most = plain_forward ? 13000 : 16384;
    auto pays = [&](int parts) {
        const int64_t w = wavefronts * parts, each = blocks / std::max<int64_t>(P->n_groups * parts, 1);      // (blocks of a part, rounded down)
        if (elem == 2) return w <= 2400 || (parts == 2 && w <= 4608 && each >= 4);
        return w <= 3072 || (w <= 6144 && each >= 2) || (parts == 2 && w <= most && each >= 4);
    };
    return pays(4) ? 4 : pays(2) ? 2 : 1;
}

// a tile in parts: one head a workgroup, so that no wavefront of it lies past the last head
inline Narrow narrow_parts(Narrow nw, int parts) {
    if (parts > 1) nw.slices = nw.heads;
    return nw;
}

constexpr int FAST_BATCH = 4;
// Wavefronts a work item for the kernels that walk single rows.  The fused kernels walk them on graphs of fewer than 1536 items (with
// row groups switched off: on any), the separate operators' SpMM where it is handed a plan without groups.  There a launch lasts
// as long as its longest item: 16 batches of four edges one after the other, each a round trip to memory.  Forward / destination
// side / source side, one -> four -> eight wavefronts an item, 8 x 64 float32 unless said otherwise, us:
//   127 items (L = 64)                  9.4 / 13.7 / 7.2  -> 4.7 / 6.4 / 4.2   -> 4.8 / 5.6 / 4.2;   SpMM 7.5 -> 4.0 -> 3.8
//   539 (L = 256, k = 16)              11.1 / 16.6 / 14.4 -> 9.2 / 11.7 / 11.6 -> 8.2 / 9.4 / 10.8;  bfloat16 12.2 / 16.9 / 15.5 -> 6.0 / 7.3 / 7.4 -> 5.6 / 6.6 / 7.4
//   816 (L = 400)                      11.4 / 16.6 / 13.8 -> 7.9 / 10.0 / 11.0 -> 9.0 / 10.4 / 10.5; SpMM 10.8 -> 6.7 -> 6.7
//   1434 (L = 700, k = 1)              15.7 / 21.2 / 15.0 -> 10.1 / 12.0 / 12.2 -> 11.3 / 12.8 / 12.6; SpMM 11.6 -> 7.9 -> 7.1
//   2050 (L = 1000, k = 1, no groups)  16.8 / 22.2 / 17.9 -> 11.0 / 14.0 / 13.6 -> 14.1 / 17.0 / 15.4; SpMM 11.6 -> 8.4 -> 8.2
// Larger launches fill the GPU with a wavefront an item.  Rows of 1024 columns take twice the registers and the LDS: eight
// wavefronts an item of them are one round of the chip up to 256 items, beyond it four are faster.  16 x 64:
//   268 (L = 130, k = 4)               16.3 / 22.7 / 16.7 -> 7.9 / 10.4 / 9.3   -> 8.2 / 10.2 / 9.4;   bfloat16 16.4 / 21.3 / 19.6 -> 7.6 / 9.6 / 8.7 -> 8.3 / 8.7 / 11.4
//   324 (L = 160, k = 4)               15.7 / 22.1 / 18.1 -> 8.5 / 10.2 / 13.1  -> 10.2 / 12.0 / 12.6; bfloat16 16.0 / 20.7 / 19.8 -> 7.6 / 9.6 / 11.5 -> 10.5 / 10.8 / 12.2
//   585 (L = 256, k = 16, both ways)   18.7 / 26.8 / 23.4 -> 18.6 / 21.2 / 19.4 -> 22.3 / 24.3 / 21.2
// A float32 forward of 512 columns or more that already has a wavefront for each of the 1024 SIMDs and 25 edges or more an
// item waits for the rate of its loads, not for one item: one -> four, 8 x 64 and 16 x 64, 983 items of 25 790 edges 11.7 -> 12.4 and 19.1 ->
// 21.0; 957 of 32 613 12.0 -> 12.2 and 19.7 -> 20.4; (1018 of 23 540 11.3 -> 11.2 and 18.2 -> 18.7; 756 items 11.2 -> 10.4 and 18.6 -> 17.1).
inline int row_parts(const bpt_plan *P, int columns, bool forward_f32 = false) {
    if (P->n_items <= (columns > 512 ? 288 : 640)) return 8;
    if (forward_f32 && columns >= 512 && P->n_items > 800 && P->n_items <= 1024 && P->n_edges >= 25000) return 1;
    return P->n_items <= 2048 ? 4 : 1;
}

}  // namespace
