// libbptblock: gfx950 kernels of what a transformer block does around its attention (C ABI in include/bptblock.h).
#include "bpttiles.h"

#include "../../include/bptblock.h"

namespace {

// ---- layer norm of a sum ------------------------------------------------------------------------------------------------------
// y = (z - mean) rstd w + b, z = x + r, and back: with g = dy w, xhat = (z - mean) rstd
//   dz = rstd (g - mean(g) - xhat mean(g xhat)),  dw = sum over the rows of dy xhat,  db = sum over the rows of dy.
// Bound by memory: the forward reads x and r and writes y, the backward reads x, r and dy and writes dz (z is formed again: storing it
// would cost the forward what the backward saves).  TPR lanes own a row and keep it in registers, NV vectors of 16 bytes each, so
// mean and variance are two passes over registers and every element is read once.  A workgroup walks rows with a stride of the grid and
// keeps weight and bias (backward: the row sums dw and db) in registers meanwhile.  dw and db: lanes -> the workgroup's rows in
// LDS -> one partial row a workgroup -> k_norm_finish, all in a fixed order.
// A last vector that would run over the row's end starts at cols - VE instead; what it repeats of its neighbour counts as 0 in the
// sums and is stored twice with one value.
// Forward / backward, us and TB/s of what they read and write: 33598 x 300 float32 24.8 (4.9) / 29.6 (5.4), 16383 x 512 float32 20.8 (4.8) / 28.8 (4.7),
// 65535 x 1024 bfloat16 84 (4.8) / 115 (4.7); k_norm_finish 4 to 5 more; a copy of 1 GiB runs at 5.0.  Workgroups of 256 threads: 16383 x 512 backward
// 28.9 -> 24.5, but 65535 x 512 98 -> 104 and at 4096 columns k_norm_finish 5 -> 11 (twice the partial rows); of 1024: slower throughout.
constexpr int NORM_BLOCK = 512;

template <typename T> struct NormElem { using acc = float; };
template <> struct NormElem<double> { using acc = double; };
template <typename T> constexpr int norm_ve() { return 16 / (int)sizeof(T); }
typedef uint32_t norm_vec16 __attribute__((ext_vector_type(4), aligned(16)));
typedef uint32_t norm_vec8 __attribute__((ext_vector_type(4), aligned(8)));
typedef uint32_t norm_vec4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t norm_vec2 __attribute__((ext_vector_type(4), aligned(2)));
template <int ALIGN> struct NormVec { typedef norm_vec16 type; };
template <> struct NormVec<8> { typedef norm_vec8 type; };
template <> struct NormVec<4> { typedef norm_vec4 type; };
template <> struct NormVec<2> { typedef norm_vec2 type; };

// VE elements from p, as 16-byte loads; AL: p lies on 16 bytes, otherwise on an element's size
template <typename T, int VE, bool AL, typename A> __device__ __forceinline__ void norm_load(const T *p, A (&out)[VE]) {
    if constexpr (VE == 1) {
        out[0] = Elem<T>::ld(p);
    } else {
        typedef typename NormVec<AL ? 16 : (int)sizeof(T)>::type vec;
        const vec w = *reinterpret_cast<const vec *>(p);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                out[2 * i] = __uint_as_float(w[i] << 16);
                out[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) out[i] = __hiloint2double((int)w[2 * i + 1], (int)w[2 * i]);
        }
    }
}
template <typename T, int VE, bool AL, typename A> __device__ __forceinline__ void norm_store(T *p, const A (&x)[VE]) {
    if constexpr (VE == 1) {
        Elem<T>::st(p, x[0]);
    } else {
        typedef typename NormVec<AL ? 16 : (int)sizeof(T)>::type vec;
        vec w;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) { w[2 * i] = (uint32_t)__double2loint(x[i]); w[2 * i + 1] = (uint32_t)__double2hiint(x[i]); }
        }
        *reinterpret_cast<vec *>(p) = w;
    }
}

// sum over the TPR lanes that own a row, in all of them (TPR > 64: the row's wavefronts meet in `meet`, two floats a wavefront and use)
template <int TPR> __device__ __forceinline__ float norm_lanes_sum(float x) {
    x = head_sum<16>(x);
    if constexpr (TPR >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if constexpr (TPR >= 64) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return x;
}
template <int TPR> __device__ __forceinline__ double norm_lanes_sum(double x) {
#pragma unroll
    for (int o = (TPR < WAVE ? TPR : WAVE) / 2; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
template <int TPR, typename A> __device__ __forceinline__ void norm_row_sum(A &x, A *meet) {
    x = norm_lanes_sum<TPR>(x);
    if constexpr (TPR > WAVE) {
        constexpr int W = TPR / WAVE;
        const int w = threadIdx.x >> 6;
        __syncthreads();                                          // (the places may still be read from the sum before)
        if ((threadIdx.x & 63) == 0) meet[w] = x;
        __syncthreads();
        const int first = w / W * W;
        x = meet[first];
#pragma unroll
        for (int i = 1; i < W; ++i) x += meet[first + i];
    }
}

// where vector i of a lane starts, and from which of its elements on it is the first to have them (VE: none, the vector lies past the end)
template <int TPR, int VE> struct NormCols {
    int at, from;
    __device__ __forceinline__ NormCols(int i, int lane, int cols) {
        const int want = (i * TPR + lane) * VE;
        at = min(want, cols - VE);
        from = min(want - at, VE);
    }
};

template <typename T, int TPR, int NV, int VE, bool AL>
__global__ __launch_bounds__(NORM_BLOCK) void k_norm_fwd(const T *__restrict__ x, const T *__restrict__ r, const T *__restrict__ w, const T *__restrict__ b,
                                                         T *__restrict__ y, typename NormElem<T>::acc *__restrict__ stats, int64_t rows, int cols,
                                                         typename NormElem<T>::acc eps) {
    using A = typename NormElem<T>::acc;
    constexpr int SLOTS = NORM_BLOCK / TPR;
    __shared__ A meet[NORM_BLOCK / WAVE];
    const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const A inv = A(1) / (A)cols;
    A wv[NV][VE], bv[NV][VE];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const NormCols<TPR, VE> c(i, lane, cols);
#pragma unroll
        for (int e = 0; e < VE; ++e) { wv[i][e] = A(1); bv[i][e] = A(0); }
        if (w) norm_load<T, VE, false>(w + c.at, wv[i]);
        if (b) norm_load<T, VE, false>(b + c.at, bv[i]);
    }
    // (every row slot of a workgroup goes round as often: the sums of rows of several wavefronts have barriers)
    for (int64_t base = (int64_t)blockIdx.x * SLOTS; base < rows; base += (int64_t)gridDim.x * SLOTS) {
        const int64_t row = base + slot;
        const bool there = row < rows;
        const int64_t off = (there ? row : rows - 1) * cols;
        A z[NV][VE];
#pragma unroll
        for (int i = 0; i < NV; ++i) norm_load<T, VE, AL>(x + off + NormCols<TPR, VE>(i, lane, cols).at, z[i]);
        if (r) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                A t[VE];
                norm_load<T, VE, AL>(r + off + NormCols<TPR, VE>(i, lane, cols).at, t);
#pragma unroll
                for (int e = 0; e < VE; ++e) z[i][e] += t[e];
            }
        }
        A sum = A(0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const NormCols<TPR, VE> c(i, lane, cols);
#pragma unroll
            for (int e = 0; e < VE; ++e) sum += e >= c.from ? z[i][e] : A(0);
        }
        norm_row_sum<TPR>(sum, meet);
        const A mean = sum * inv;
        sum = A(0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const NormCols<TPR, VE> c(i, lane, cols);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                z[i][e] -= mean;
                sum += e >= c.from ? z[i][e] * z[i][e] : A(0);
            }
        }
        norm_row_sum<TPR>(sum, meet);
        const A rstd = A(1) / sqrt(sum * inv + eps);
        if (!there) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const NormCols<TPR, VE> c(i, lane, cols);
#pragma unroll
            for (int e = 0; e < VE; ++e) z[i][e] = z[i][e] * rstd * wv[i][e] + bv[i][e];
            if (c.from < VE) norm_store<T, VE, AL>(y + off + c.at, z[i]);
        }
        if (stats && lane == 0) {
            stats[2 * row] = mean;
            stats[2 * row + 1] = rstd;
        }
    }
}

// part: (gridDim.x, 2, cols) partial sums of dw and db, or null (then the workgroup's own go to dw and db: a grid of one)
template <typename T, int TPR, int NV, int VE, bool AL>
__global__ __launch_bounds__(NORM_BLOCK) void k_norm_bwd(const T *__restrict__ x, const T *__restrict__ r, const T *__restrict__ w,
                                                         const typename NormElem<T>::acc *__restrict__ stats, const T *__restrict__ dy, T *__restrict__ dz,
                                                         typename NormElem<T>::acc *__restrict__ part, T *__restrict__ dw, T *__restrict__ db,
                                                         int64_t rows, int cols) {
    using A = typename NormElem<T>::acc;
    constexpr int SLOTS = NORM_BLOCK / TPR, PER_WAVE = TPR < WAVE ? WAVE / TPR : 1;
    __shared__ A meet[NORM_BLOCK / WAVE][2];
    const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const A inv = A(1) / (A)cols;
    A wv[NV][VE], sw[NV][VE], sb[NV][VE];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < VE; ++e) { wv[i][e] = A(1); sw[i][e] = sb[i][e] = A(0); }
        if (w) norm_load<T, VE, false>(w + NormCols<TPR, VE>(i, lane, cols).at, wv[i]);
    }
    for (int64_t base = (int64_t)blockIdx.x * SLOTS; base < rows; base += (int64_t)gridDim.x * SLOTS) {
        const int64_t row = base + slot;
        const bool there = row < rows;
        const int64_t off = (there ? row : rows - 1) * cols;
        const int64_t at = 2 * (there ? row : rows - 1);
        const A mean = stats ? stats[at] : A(0), rstd = stats ? stats[at + 1] : A(1);
        A z[NV][VE], g[NV][VE];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const NormCols<TPR, VE> c(i, lane, cols);
            norm_load<T, VE, AL>(x + off + c.at, z[i]);
            norm_load<T, VE, AL>(dy + off + c.at, g[i]);
        }
        if (r) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                A t[VE];
                norm_load<T, VE, AL>(r + off + NormCols<TPR, VE>(i, lane, cols).at, t);
#pragma unroll
                for (int e = 0; e < VE; ++e) z[i][e] += t[e];
            }
        }
        A s0 = A(0), s1 = A(0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const NormCols<TPR, VE> c(i, lane, cols);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const bool mine = there && e >= c.from;
                z[i][e] = (z[i][e] - mean) * rstd;
                sw[i][e] += mine ? g[i][e] * z[i][e] : A(0);
                sb[i][e] += mine ? g[i][e] : A(0);
                g[i][e] *= wv[i][e];
                s0 += mine ? g[i][e] : A(0);
                s1 += mine ? g[i][e] * z[i][e] : A(0);
            }
        }
        if (!dz) continue;
        s0 = norm_lanes_sum<TPR>(s0);
        s1 = norm_lanes_sum<TPR>(s1);
        if constexpr (TPR > WAVE) {
            constexpr int W = TPR / WAVE;
            const int wv_ = threadIdx.x >> 6, first = wv_ / W * W;
            __syncthreads();
            if ((threadIdx.x & 63) == 0) { meet[wv_][0] = s0; meet[wv_][1] = s1; }
            __syncthreads();
            s0 = meet[first][0];
            s1 = meet[first][1];
#pragma unroll
            for (int i = 1; i < W; ++i) { s0 += meet[first + i][0]; s1 += meet[first + i][1]; }
        }
        if (!there) continue;
        s0 *= inv;
        s1 *= inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const NormCols<TPR, VE> c(i, lane, cols);
#pragma unroll
            for (int e = 0; e < VE; ++e) g[i][e] = rstd * (g[i][e] - s0 - z[i][e] * s1);
            if (c.from < VE) norm_store<T, VE, AL>(dz + off + c.at, g[i]);
        }
    }
    if (!dw && !db && !part) return;
    // rows of one wavefront by lane, then the workgroup's rows in LDS: [row of the workgroup][column], dw first, then db
    constexpr int GROUPS = TPR < WAVE ? NORM_BLOCK / WAVE : SLOTS;
    constexpr int COLS = TPR * NV * VE;
    __shared__ A sums[GROUPS][COLS];
    const int group = TPR < WAVE ? threadIdx.x >> 6 : slot;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                A v = which == 0 ? sw[i][e] : sb[i][e];
                if constexpr (PER_WAVE > 1) {
#pragma unroll
                    for (int o = TPR; o < WAVE; o <<= 1) v += __shfl_xor(v, o);
                }
                if (PER_WAVE == 1 || (threadIdx.x & 63) < TPR) sums[group][(i * TPR + lane) * VE + e] = v;
            }
        }
        __syncthreads();
        // (a column of a last vector that starts early sits where that vector would have started)
        for (int c = threadIdx.x; c < cols; c += NORM_BLOCK) {
            const int tail = cols % VE, at = VE > 1 && tail != 0 && c >= cols - tail ? (cols - tail) + (c - (cols - VE)) : c;
            A v = A(0);
#pragma unroll
            for (int k = 0; k < GROUPS; ++k) v += sums[k][at];
            if (part) part[((int64_t)blockIdx.x * 2 + which) * cols + c] = v;
            else if (which == 0 && dw) Elem<T>::st(dw + c, v);
            else if (which == 1 && db) Elem<T>::st(db + c, v);
        }
    }
}

// dw and db from the workgroups' partial sums: 16 columns a workgroup, sixteen lanes a column take partial p, p + 16, ...; the sixteen are
// added in their order
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_norm_finish(const typename NormElem<T>::acc *__restrict__ part, int n_parts, T *__restrict__ dw, T *__restrict__ db,
                                                       int cols) {
    using A = typename NormElem<T>::acc;
    __shared__ A meet[16][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    const int64_t at = (int64_t)blockIdx.x * 16 + c;              // column of the (2, cols) result
    A v = A(0);
    if (at < 2 * (int64_t)cols) {
        int p = k;
        for (; p + 7 * 16 < n_parts; p += 8 * 16) {
            A t[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) t[u] = part[(int64_t)(p + u * 16) * 2 * cols + at];
#pragma unroll
            for (int u = 0; u < 8; ++u) v += t[u];
        }
        for (; p < n_parts; p += 16) v += part[(int64_t)p * 2 * cols + at];
    }
    meet[k][c] = v;
    __syncthreads();
    if (k != 0 || at >= 2 * (int64_t)cols) return;
    v = meet[0][c];
#pragma unroll
    for (int i = 1; i < 16; ++i) v += meet[i][c];
    T *const out = at < cols ? dw : db;
    if (out) Elem<T>::st(out + (at < cols ? at : at - cols), v);
}

// Rows too long for a workgroup's registers: a workgroup a row, three walks over it (the second and third come from the caches).
template <typename A> __device__ __forceinline__ A norm_block_sum(A x, A *meet) {
    x = norm_lanes_sum<WAVE>(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) meet[threadIdx.x >> 6] = x;
    __syncthreads();
    A s = meet[0];
#pragma unroll
    for (int i = 1; i < NORM_BLOCK / WAVE; ++i) s += meet[i];
    return s;
}
template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void k_norm_fwd_long(const T *__restrict__ x, const T *__restrict__ r, const T *__restrict__ w,
                                                              const T *__restrict__ b, T *__restrict__ y, typename NormElem<T>::acc *__restrict__ stats,
                                                              int64_t cols, typename NormElem<T>::acc eps) {
    using A = typename NormElem<T>::acc;
    __shared__ A meet[NORM_BLOCK / WAVE];
    const int64_t off = (int64_t)blockIdx.x * cols;
    auto z = [&](int64_t c) { const A v = Elem<T>::ld(x + off + c); return r ? v + (A)Elem<T>::ld(r + off + c) : v; };
    A s = A(0);
    for (int64_t c = threadIdx.x; c < cols; c += NORM_BLOCK) s += z(c);
    const A mean = norm_block_sum(s, meet) / (A)cols;
    s = A(0);
    for (int64_t c = threadIdx.x; c < cols; c += NORM_BLOCK) { const A v = z(c) - mean; s += v * v; }
    const A rstd = A(1) / sqrt(norm_block_sum(s, meet) / (A)cols + eps);
    for (int64_t c = threadIdx.x; c < cols; c += NORM_BLOCK)
        Elem<T>::st(y + off + c, (z(c) - mean) * rstd * (w ? (A)Elem<T>::ld(w + c) : A(1)) + (b ? (A)Elem<T>::ld(b + c) : A(0)));
    if (stats && threadIdx.x == 0) {
        stats[2 * (int64_t)blockIdx.x] = mean;
        stats[2 * (int64_t)blockIdx.x + 1] = rstd;
    }
}
template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void k_norm_bwd_long(const T *__restrict__ x, const T *__restrict__ r, const T *__restrict__ w,
                                                              const typename NormElem<T>::acc *__restrict__ stats, const T *__restrict__ dy, T *__restrict__ dz,
                                                              int64_t cols) {
    using A = typename NormElem<T>::acc;
    __shared__ A meet[NORM_BLOCK / WAVE];
    const int64_t off = (int64_t)blockIdx.x * cols;
    const A mean = stats[2 * (int64_t)blockIdx.x], rstd = stats[2 * (int64_t)blockIdx.x + 1];
    auto xhat = [&](int64_t c) { const A v = Elem<T>::ld(x + off + c); return ((r ? v + (A)Elem<T>::ld(r + off + c) : v) - mean) * rstd; };
    auto g = [&](int64_t c) { return (A)Elem<T>::ld(dy + off + c) * (w ? (A)Elem<T>::ld(w + c) : A(1)); };
    A s0 = A(0), s1 = A(0);
    for (int64_t c = threadIdx.x; c < cols; c += NORM_BLOCK) { const A v = g(c); s0 += v; s1 += v * xhat(c); }
    s0 = norm_block_sum(s0, meet) / (A)cols;
    s1 = norm_block_sum(s1, meet) / (A)cols;
    for (int64_t c = threadIdx.x; c < cols; c += NORM_BLOCK) Elem<T>::st(dz + off + c, rstd * (g(c) - s0 - xhat(c) * s1));
}
// partial sums of dw and db, a column a thread: workgroup (strip of NORM_BLOCK columns, part) walks the rows part, part + parts, ...
template <typename T>
__global__ __launch_bounds__(NORM_BLOCK) void k_norm_sums_long(const T *__restrict__ x, const T *__restrict__ r, const typename NormElem<T>::acc *__restrict__ stats,
                                                               const T *__restrict__ dy, typename NormElem<T>::acc *__restrict__ part, int64_t rows, int64_t cols) {
    using A = typename NormElem<T>::acc;
    const int64_t c = (int64_t)blockIdx.x * NORM_BLOCK + threadIdx.x;
    if (c >= cols) return;
    A sw = A(0), sb = A(0);
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const A mean = stats ? stats[2 * row] : A(0), rstd = stats ? stats[2 * row + 1] : A(1), g = Elem<T>::ld(dy + row * cols + c);
        A v = Elem<T>::ld(x + row * cols + c);
        if (r) v += (A)Elem<T>::ld(r + row * cols + c);
        sw += g * ((v - mean) * rstd);
        sb += g;
    }
    part[((int64_t)blockIdx.y * 2) * cols + c] = sw;
    part[((int64_t)blockIdx.y * 2 + 1) * cols + c] = sb;
}

// workgroups that walk rows: two a compute unit (four: 16383 x 512 backward 28.9 -> 35.9 us, the partial rows are a sixteenth of its bytes then)
constexpr int NORM_PARTS = 512, NORM_PARTS_LONG = 64;

// lanes a row and vectors a lane: the least room, and of equal room the most vectors (fewer steps to add lanes up)
struct NormShape { int tpr, nv; };           // tpr 0: rows too long
inline NormShape norm_shape(int64_t cols, int ve) {
    const int64_t need = (cols + ve - 1) / ve;
    NormShape best{0, 0};
    for (int tpr : {16, 32, 64, 256})
        for (int nv : {4, 3, 2, 1})
            if ((int64_t)tpr * nv >= need && (best.tpr == 0 || tpr * nv < best.tpr * best.nv)) best = NormShape{tpr, nv};
    return best;
}
template <typename T> inline int64_t norm_longest() { return (int64_t)256 * 4 * norm_ve<T>(); }
template <typename T> inline int norm_parts(int64_t rows, int64_t cols) {
    if (cols > norm_longest<T>()) return (int)std::min<int64_t>(NORM_PARTS_LONG, std::max<int64_t>(rows, 1));
    const NormShape s = norm_shape(cols, cols < norm_ve<T>() ? 1 : norm_ve<T>());
    const int64_t slots = NORM_BLOCK / s.tpr;
    // one workgroup, no partial sums, one launch less: 512 columns float32 (16 slots), backward with and without, 32 rows 7.0 / 8.4 us, 64 rows 10.0 / 8.4
    if (rows <= 2 * slots) return 1;
    return (int)std::min<int64_t>(NORM_PARTS, std::max<int64_t>((rows + slots - 1) / slots, 1));
}

inline bool on16(std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if (p && !aligned16(p)) return false;
    return true;
}

// F(tpr, nv, ve, al) with compile-time values
template <typename T, typename F> int norm_pick(int64_t cols, bool al, F &&f) {
    constexpr int VE = norm_ve<T>();
    using std::integral_constant;
#define GO(TP, N, V, ALIGNED) return f(integral_constant<int, TP>{}, integral_constant<int, N>{}, integral_constant<int, V>{}, integral_constant<bool, ALIGNED>{})
    if (cols < VE) GO(16, 1, 1, false);
    const NormShape s = norm_shape(cols, VE);
#define ROW(TP, N) \
    if (s.tpr == TP && s.nv == N) { if (al) GO(TP, N, VE, true); else GO(TP, N, VE, false); }
#define ROWS(TP) ROW(TP, 1) ROW(TP, 2) ROW(TP, 3) ROW(TP, 4)
    ROWS(16) ROWS(32) ROWS(64) ROWS(256)
#undef ROWS
#undef ROW
#undef GO
    return BPT_ERR_SHAPE;
}

template <typename T>
int run_norm_fwd(const void *x_, const void *r_, const void *w_, const void *b_, void *y_, void *stats_, int64_t rows, int64_t cols, double eps, hipStream_t s) {
    using A = typename NormElem<T>::acc;
    const T *x = (const T *)x_, *r = (const T *)r_, *w = (const T *)w_, *b = (const T *)b_;
    T *y = (T *)y_;
    A *stats = (A *)stats_;
    if (rows == 0) return BPT_OK;
    if (cols > norm_longest<T>()) {
        hipLaunchKernelGGL((k_norm_fwd_long<T>), dim3((unsigned)rows), dim3(NORM_BLOCK), 0, s, x, r, w, b, y, stats, cols, (A)eps);
        return launch_status();
    }
    return norm_pick<T>(cols, cols % norm_ve<T>() == 0 && on16({x, r, y}), [&](auto tpr, auto nv, auto ve, auto al) {
        constexpr int SLOTS = NORM_BLOCK / tpr();
        const int64_t blocks = std::min<int64_t>((rows + SLOTS - 1) / SLOTS, 4 * NORM_PARTS);
        hipLaunchKernelGGL((k_norm_fwd<T, tpr(), nv(), ve(), al()>), dim3((unsigned)blocks), dim3(NORM_BLOCK), 0, s, x, r, w, b, y, stats, rows, (int)cols, (A)eps);
        return launch_status();
    });
}

template <typename T>
int run_norm_bwd(const void *x_, const void *r_, const void *w_, const void *stats_, const void *dy_, void *dz_, void *dw_, void *db_, void *ws, int64_t rows,
                 int64_t cols, hipStream_t s) {
    using A = typename NormElem<T>::acc;
    const T *x = (const T *)x_, *r = (const T *)r_, *w = (const T *)w_, *dy = (const T *)dy_;
    const A *stats = (const A *)stats_;
    T *dz = (T *)dz_, *dw = (T *)dw_, *db = (T *)db_;
    A *part = (A *)ws;
    const bool sums = dw || db;
    if (!sums && (!dz || rows == 0)) return BPT_OK;
    int parts = rows == 0 ? 0 : norm_parts<T>(rows, cols);
    if (rows > 0 && cols > norm_longest<T>()) {
        if (dz) hipLaunchKernelGGL((k_norm_bwd_long<T>), dim3((unsigned)rows), dim3(NORM_BLOCK), 0, s, x, r, w, stats, dy, dz, cols);
        if (sums)
            hipLaunchKernelGGL((k_norm_sums_long<T>), dim3((unsigned)((cols + NORM_BLOCK - 1) / NORM_BLOCK), parts), dim3(NORM_BLOCK), 0, s, x, r, stats, dy, part,
                               rows, cols);
    } else if (rows > 0) {
        const bool alone = parts == 1;                            // one workgroup has the sums whole
        const int st = norm_pick<T>(cols, cols % norm_ve<T>() == 0 && on16({x, r, dy, dz}), [&](auto tpr, auto nv, auto ve, auto al) {
            hipLaunchKernelGGL((k_norm_bwd<T, tpr(), nv(), ve(), al()>), dim3((unsigned)parts), dim3(NORM_BLOCK), 0, s, x, r, w, stats, dy, dz,
                               sums && !alone ? part : nullptr, alone ? dw : nullptr, alone ? db : nullptr, rows, (int)cols);
            return launch_status();
        });
        if (st != BPT_OK || alone) return st;
    }
    const int st = launch_status();
    if (st != BPT_OK || !sums) return st;
    hipLaunchKernelGGL((k_norm_finish<T>), dim3((unsigned)((2 * cols + 15) / 16)), dim3(BLOCK), 0, s, part, parts, dw, db, (int)cols);
    return launch_status();
}

// ---- relu kept in 8 bits -----------------------------------------------------------------------------------------------------
// What a feed-forward's backward needs of relu's result is its value in one product (the second layer's weight gradient) and its sign.
// 64 neighbouring activations share a step 2^e, the smallest power of two with 255 steps up to their largest, and an activation is
// a whole number of steps in one byte: off by half a step at most, 2^-8 of the block's largest (a step that is a power of two costs up
// to one bit against amax / 255, and makes scaling, rounding and the value read back exact in both types).  A positive activation
// keeps a step at least, so the byte also is the mask of relu and of dropout.
// Bound by memory: the forward reads a and writes y and 1 + 1/64 bytes, the backward reads dy and those and writes da and y8.  A lane has 16
// bytes of a, so a block is 16 (float32) or 8 (bfloat16) neighbouring lanes, whose maximum takes four or three DPP steps.
// Forward / backward, us and TB/s of what they read and write: 1023 x 2048 float32 6.4 / 6.4 (in the caches), 16383 x 2048 float32 58 (5.2) / 75 (5.8),
// 65535 x 4096 bfloat16 241 (5.6) / 341 (5.5).
template <int LANES> __device__ __forceinline__ float lanes_max(float x) {
    x = fmaxf(x, dpp_mov<0xB1>(x));
    x = fmaxf(x, dpp_mov<0x4E>(x));
    x = fmaxf(x, dpp_mov<0x141>(x));
    if constexpr (LANES >= 16) x = fmaxf(x, dpp_mov<0x140>(x));
    return x;
}
// the smallest e >= -126 with top <= 255 2^e, top finite and not negative: top = m 2^x, m in [1, 2), is within 255 2^(x - 7) = (255 / 128) 2^x or not
__device__ __forceinline__ int relu8_exp(float top) {
    const uint32_t u = __float_as_uint(top);
    return max((int)(u >> 23) - 127 - 7 + ((u & 0x7fffffu) > 0x7f0000u ? 1 : 0), -126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }          // -126 <= e <= 127

constexpr int RELU8_UNROLL = 4;
typedef uint32_t relu8_word1 __attribute__((ext_vector_type(1)));
typedef uint32_t relu8_word2 __attribute__((ext_vector_type(2)));
template <int VE> struct Relu8Word { typedef relu8_word1 type; };      // the codes of a lane's vector
template <> struct Relu8Word<8> { typedef relu8_word2 type; };

template <typename T, bool AL, bool DROP>
__global__ __launch_bounds__(BLOCK) void k_relu8_fwd(const T *__restrict__ a, T *__restrict__ y, uint8_t *__restrict__ codes, int8_t *__restrict__ exps, int64_t n,
                                                     uint32_t drop_thr, uint32_t drop_seed, float drop_inv) {
    constexpr int VE = norm_ve<T>(), LANES = BPT_RELU8_BLOCK / VE;
    typedef typename Relu8Word<VE>::type word;
    const int64_t first = ((int64_t)blockIdx.x * RELU8_UNROLL * BLOCK + threadIdx.x) * VE;
    float x[RELU8_UNROLL][VE];
#pragma unroll
    for (int u = 0; u < RELU8_UNROLL; ++u) {
        const int64_t at = first + (int64_t)u * BLOCK * VE;
        if (at + VE <= n) {
            norm_load<T, VE, AL>(a + at, x[u]);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) x[u][e] = at + e < n ? (float)Elem<T>::ld(a + at + e) : 0.f;
        }
    }
    issue_loads_first();
#pragma unroll
    for (int u = 0; u < RELU8_UNROLL; ++u) {
        const int64_t at = first + (int64_t)u * BLOCK * VE;
        float top = 0.f;
        bool odd = false;                                         // something infinite or NaN
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            float v = x[u][e] <= 0.f ? 0.f : x[u][e];              // (NaN stays)
            if constexpr (DROP) {
                v = dropout_keep((uint32_t)(at + e), drop_seed, drop_thr, drop_inv) != 0.f ? v * drop_inv : 0.f;
                if constexpr (sizeof(T) == 2) v = __uint_as_float(pack_bf16(v, v) << 16);        // (the step goes by what is stored)
            }
            x[u][e] = v;
            odd |= !(v < INFINITY);
            top = fmaxf(top, v);
        }
        top = lanes_max<LANES>(odd ? INFINITY : top);
        const bool finite = top < INFINITY;
        const int ex = finite ? relu8_exp(top) : BPT_RELU8_NAN;
        const float steps = finite ? pow2(-ex) : 0.f;
        uint32_t code[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float v = x[u][e];
            code[e] = v == 0.f ? 0u : finite ? max((uint32_t)rintf(v * steps), 1u) : 1u;
        }
        if (at + VE <= n) {
            if (y) norm_store<T, VE, AL>(y + at, x[u]);
            word c;
#pragma unroll
            for (int i = 0; i < VE / 4; ++i) c[i] = code[4 * i] | code[4 * i + 1] << 8 | code[4 * i + 2] << 16 | code[4 * i + 3] << 24;
            *reinterpret_cast<word *>(codes + at) = c;
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (at + e < n) {
                    if (y) Elem<T>::st(y + at + e, x[u][e]);
                    codes[at + e] = (uint8_t)code[e];
                }
        }
        if (at < n && threadIdx.x % LANES == 0) exps[at / BPT_RELU8_BLOCK] = (int8_t)ex;
    }
}

template <typename T, bool AL>
__global__ __launch_bounds__(BLOCK) void k_relu8_bwd(const T *dy, const uint8_t *__restrict__ codes, const int8_t *__restrict__ exps, T *da,
                                                     T *__restrict__ y8, int64_t n, float drop_inv) {
    constexpr int VE = norm_ve<T>();
    typedef typename Relu8Word<VE>::type word;
    const int64_t first = ((int64_t)blockIdx.x * RELU8_UNROLL * BLOCK + threadIdx.x) * VE;
    float g[RELU8_UNROLL][VE];
    word c[RELU8_UNROLL];
    int ex[RELU8_UNROLL];
#pragma unroll
    for (int u = 0; u < RELU8_UNROLL; ++u) {
        const int64_t at = first + (int64_t)u * BLOCK * VE;
        ex[u] = at < n ? exps[at / BPT_RELU8_BLOCK] : 0;
        if (at + VE <= n) {
            c[u] = *reinterpret_cast<const word *>(codes + at);
            if (da) norm_load<T, VE, AL>(dy + at, g[u]);
        } else {
#pragma unroll
            for (int i = 0; i < VE / 4; ++i) c[u][i] = 0;
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                g[u][e] = 0.f;
                if (at + e < n) {
                    c[u][e / 4] |= (uint32_t)codes[at + e] << 8 * (e % 4);
                    if (da) g[u][e] = Elem<T>::ld(dy + at + e);
                }
            }
        }
    }
    issue_loads_first();
#pragma unroll
    for (int u = 0; u < RELU8_UNROLL; ++u) {
        const int64_t at = first + (int64_t)u * BLOCK * VE;
        const float step = ex[u] == BPT_RELU8_NAN ? NAN : pow2(ex[u]);
        float v[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const uint32_t code = c[u][e / 4] >> 8 * (e % 4) & 255u;
            v[e] = code == 0u ? 0.f : (float)code * step;
            g[u][e] = code == 0u ? 0.f : g[u][e] * drop_inv;
        }
        if (at + VE <= n) {
            if (da) norm_store<T, VE, AL>(da + at, g[u]);
            if (y8) norm_store<T, VE, AL>(y8 + at, v);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (at + e < n) {
                    if (da) Elem<T>::st(da + at + e, g[u][e]);
                    if (y8) Elem<T>::st(y8 + at + e, v[e]);
                }
        }
    }
}

inline int64_t relu8_blocks(int64_t n, int ve) { return (n + (int64_t)BLOCK * RELU8_UNROLL * ve - 1) / ((int64_t)BLOCK * RELU8_UNROLL * ve); }

template <typename T> int run_relu8_fwd(const void *a, void *y, uint8_t *codes, int8_t *exps, int64_t n, Dropout drop, hipStream_t s) {
    const unsigned blocks = (unsigned)relu8_blocks(n, norm_ve<T>());
    const bool al = on16({a, y});
#define LAUNCH(AL, DR) \
    hipLaunchKernelGGL((k_relu8_fwd<T, AL, DR>), dim3(blocks), dim3(BLOCK), 0, s, (const T *)a, (T *)y, codes, exps, n, drop.thr, drop.seed, drop.inv)
    if (drop.thr != 0) { if (al) LAUNCH(true, true); else LAUNCH(false, true); }
    else { if (al) LAUNCH(true, false); else LAUNCH(false, false); }
#undef LAUNCH
    return launch_status();
}
template <typename T> int run_relu8_bwd(const void *dy, const uint8_t *codes, const int8_t *exps, void *da, void *y8, int64_t n, float inv, hipStream_t s) {
    const unsigned blocks = (unsigned)relu8_blocks(n, norm_ve<T>());
#define LAUNCH(AL) hipLaunchKernelGGL((k_relu8_bwd<T, AL>), dim3(blocks), dim3(BLOCK), 0, s, (const T *)dy, codes, exps, (T *)da, (T *)y8, n, inv)
    if (on16({da ? dy : nullptr, da, y8})) LAUNCH(true);
    else LAUNCH(false);
#undef LAUNCH
    return launch_status();
}

inline int check_norm(int64_t rows, int64_t cols, int dtype) {
    if (dtype != BPT_F32 && dtype != BPT_F64 && dtype != BPT_BF16) return BPT_ERR_DTYPE;
    if (rows < 0 || rows > 0x7fffffff || cols < 1 || cols > 0x3fffffff) return BPT_ERR_SIZE;
    return BPT_OK;
}
inline int check_relu8(int64_t n, float p, int dtype) {
    if (dtype != BPT_F32 && dtype != BPT_BF16) return BPT_ERR_DTYPE;
    if (n < 0 || n > (int64_t)1 << 40 || !(p >= 0.f && p < 1.f) || (p > 0.f && n > (int64_t)1 << 32)) return BPT_ERR_SIZE;
    return BPT_OK;
}

}  // namespace

extern "C" {

int bpt_add_norm_forward(const void *x, const void *residual, const void *weight, const void *bias, void *y, void *stats, int64_t rows, int64_t cols, double eps,
                         int dtype, void *stream) {
    const int bad = check_norm(rows, cols, dtype);
    if (bad != BPT_OK) return bad;
    if (rows > 0 && (!x || !y)) return BPT_ERR_NULL;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == BPT_F32) return run_norm_fwd<float>(x, residual, weight, bias, y, stats, rows, cols, eps, s);
    if (dtype == BPT_F64) return run_norm_fwd<double>(x, residual, weight, bias, y, stats, rows, cols, eps, s);
    return run_norm_fwd<bf16_t>(x, residual, weight, bias, y, stats, rows, cols, eps, s);
}

int64_t bpt_add_norm_workspace_bytes(int64_t rows, int64_t cols, int dtype) {
    if (check_norm(rows, cols, dtype) != BPT_OK) return -1;
    const int parts = dtype == BPT_F32 ? norm_parts<float>(rows, cols) : dtype == BPT_F64 ? norm_parts<double>(rows, cols) : norm_parts<bf16_t>(rows, cols);
    return (int64_t)parts * 2 * cols * (int64_t)acc_size(dtype);
}

int bpt_add_norm_backward(const void *x, const void *residual, const void *weight, const void *stats, const void *dy, void *dz, void *dweight, void *dbias,
                          void *workspace, int64_t workspace_bytes, int64_t rows, int64_t cols, int dtype, void *stream) {
    const int bad = check_norm(rows, cols, dtype);
    if (bad != BPT_OK) return bad;
    if (rows > 0 && (!x || !dy || (!stats && (dz || dweight)))) return BPT_ERR_NULL;
    if ((dweight || dbias) && (!workspace || workspace_bytes < bpt_add_norm_workspace_bytes(rows, cols, dtype) || !aligned16(workspace))) return BPT_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == BPT_F32) return run_norm_bwd<float>(x, residual, weight, stats, dy, dz, dweight, dbias, workspace, rows, cols, s);
    if (dtype == BPT_F64) return run_norm_bwd<double>(x, residual, weight, stats, dy, dz, dweight, dbias, workspace, rows, cols, s);
    return run_norm_bwd<bf16_t>(x, residual, weight, stats, dy, dz, dweight, dbias, workspace, rows, cols, s);
}

int bpt_relu8_forward(const void *a, void *y, uint8_t *codes, int8_t *exps, int64_t n, float dropout_p, uint64_t dropout_seed, int dtype, void *stream) {
    const int bad = check_relu8(n, dropout_p, dtype);
    if (bad != BPT_OK) return bad;
    if (n == 0) return BPT_OK;
    if (!a || !codes || !exps) return BPT_ERR_NULL;
    if (!aligned16(codes)) return BPT_ERR_UNSUPPORTED;
    const Dropout drop = make_dropout(dropout_p, dropout_seed);
    hipStream_t s = (hipStream_t)stream;
    return dtype == BPT_F32 ? run_relu8_fwd<float>(a, y, codes, exps, n, drop, s) : run_relu8_fwd<bf16_t>(a, y, codes, exps, n, drop, s);
}

int bpt_relu8_backward(const void *dy, const uint8_t *codes, const int8_t *exps, void *da, void *y8, int64_t n, float dropout_p, int dtype, void *stream) {
    const int bad = check_relu8(n, dropout_p, dtype);
    if (bad != BPT_OK) return bad;
    if (n == 0 || (!da && !y8)) return BPT_OK;
    if (!codes || !exps || (da && !dy)) return BPT_ERR_NULL;
    if (!aligned16(codes)) return BPT_ERR_UNSUPPORTED;
    const float inv = make_dropout(dropout_p, 0).inv;
    hipStream_t s = (hipStream_t)stream;
    return dtype == BPT_F32 ? run_relu8_bwd<float>(dy, codes, exps, da, y8, n, inv, s) : run_relu8_bwd<bf16_t>(dy, codes, exps, da, y8, n, inv, s);
}

}  // extern "C"
