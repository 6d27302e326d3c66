// libbptlinear: gfx950 kernels of matrix products with an epilogue and of dropout from a counter-based generator (C ABI in include/bptlinear.h).
#include "bpttiles.h"

#include "../../include/bptlinear.h"

namespace {

// ---- elements ------------------------------------------------------------------------------------------------------------------
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4_on4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t uintx4_on2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t uintx2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
template <typename T> struct Raw { typedef uint32_t type; typedef uintx4_on4 vec; };
template <> struct Raw<bf16_t> { typedef uint16_t type; typedef uintx4_on2 vec; };

template <typename T> constexpr int ve() { return 16 / (int)sizeof(T); }       // elements of 16 bytes

// four neighbouring elements, on a multiple of their size
__device__ __forceinline__ floatx4 load4(const float *p) { return *reinterpret_cast<const floatx4 *>(p); }
__device__ __forceinline__ floatx4 load4(const bf16_t *p) {
    const uintx2v w = *reinterpret_cast<const uintx2v *>(p);
    return floatx4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16), __uint_as_float(w[1] & 0xffff0000u)};
}
__device__ __forceinline__ void store4(float *p, floatx4 v) { *reinterpret_cast<floatx4 *>(p) = v; }
__device__ __forceinline__ void store4(bf16_t *p, floatx4 v) { *reinterpret_cast<uintx2v *>(p) = uintx2v{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])}; }

// ---- Philox-4x32-10 --------------------------------------------------------------------------------------------------------------
// A word an element, four elements a counter.  Ten rounds are twenty 64-bit products a counter, a quarter of the vector units' rate each.
struct Drop {
    uint32_t thr, k0, k1;        // thr 0: nothing is dropped
    float inv;
};
inline Drop make_drop(double p, uint64_t seed) {
    if (!(p > 0.0)) return Drop{0u, 0u, 0u, 1.f};
    const double t = p * 4294967296.0;                            // (its whole part counts)
    return Drop{(uint32_t)(t >= 4294967295.0 ? 4294967295.0 : t < 1.0 ? 1.0 : t), (uint32_t)seed, (uint32_t)(seed >> 32), (float)(1.0 / (1.0 - p))};
}
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
__device__ __forceinline__ uintx4 philox(uint64_t counter, uint32_t k0, uint32_t k1) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0u, c3 = 0u;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = xor3((uint32_t)(q >> 32), c1, k0);
        c1 = (uint32_t)q;
        c2 = xor3((uint32_t)(p >> 32), c3, k1);
        c3 = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return uintx4{c0, c1, c2, c3};
}
// the words of elements at .. at + 3: those of one counter, or of two where at is no multiple of 4
__device__ __forceinline__ uintx4 drop_words(uint64_t at, const Drop &d) {
    const uintx4 a = philox(at >> 2, d.k0, d.k1);
    const int s = (int)at & 3;
    if (s == 0) return a;
    const uintx4 b = philox((at >> 2) + 1, d.k0, d.k1);
    return s == 1 ? uintx4{a[1], a[2], a[3], b[0]} : s == 2 ? uintx4{a[2], a[3], b[0], b[1]} : uintx4{a[3], b[0], b[1], b[2]};
}
// (a choice, not a product: a dropped infinity is 0)
__device__ __forceinline__ floatx4 dropped(floatx4 v, uintx4 words, const Drop &d) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = words[e] >= d.thr ? v[e] * d.inv : 0.f;
    return v;
}

// ---- activations -------------------------------------------------------------------------------------------------------------------
// Phi(a) = erfc(-a / sqrt 2) / 2 from e = exp(-a^2 / 2): erfc(z) exp(z^2) = t P(t), t = 1 / (1 + 0.45 z) for z >= 0, P of degree 9 fitted to 1.6e-8 of it (least squares
// on 4000 points, weights raised where the error is largest); with the roundings of float32 2e-7 off at most.  Relative to itself, below zero, where 1 + erf keeps no digits: 4e-7 down to
// -1, 9e-7 to -4, 2e-6 to -6, 8e-6 to -13 (exp2 takes a square that has been rounded); it ends in 0 behind, where it is no normal number any more.
__device__ __forceinline__ float gaussian(float a) { return __builtin_amdgcn_exp2f(a * a * -0.72134752044448170f); }
__device__ __forceinline__ float normal_cdf(float a, float e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(a), 0.45f * 0.70710678118654752f, 1.f));
    constexpr float P[10] = {0.253877291f,  0.254068526f,  0.226492773f,  0.184594003f, 0.0902296561f,
                             0.0373546171f, 0.0662443061f, -0.240835511f, 0.164408172f, -0.0364338496f};
    float p = P[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) p = fmaf(p, t, P[i]);
    p *= 0.5f * t * e;
    return a < 0.f ? p : 1.f - p;                                 // (NaN: 1 - NaN)
}
__device__ __forceinline__ float activated(float a, int act) {
    if (act == BPT_ACT_RELU) return a <= 0.f ? 0.f : a;           // (NaN stays)
    if (act == BPT_ACT_GELU) return a * normal_cdf(a, gaussian(a));
    return a;
}
// g act'(a)
__device__ __forceinline__ float activated_back(float g, float a, int act) {
    if (act == BPT_ACT_RELU) return a <= 0.f ? 0.f : g;
    if (act == BPT_ACT_GELU) {
        const float e = gaussian(a);
        return g * fmaf(a * e, 0.39894228040143268f, normal_cdf(a, e));
    }
    return g;
}

// What follows a product: four neighbouring columns of a row at a time.
template <typename T> struct Epilogue {
    const T *bias, *residual;
    T *y, *kept;
    int64_t cols;
    float scale;                 // of the product
    int act;
    Drop drop;
    bool quads;                  // rows, and with them quads, start on four elements everywhere
    // four columns, of rows that start on four, of an activation and dropout that the caller has looked up; bias of the columns, residual as read ahead; a is kept of an activation
    template <int ACT, bool DROP> __device__ __forceinline__ void quad(floatx4 v, int64_t at, floatx4 b, floatx4 ahead) const {
        v = v * scale + b;
        if constexpr (ACT != BPT_ACT_NONE) {
            if (kept) store4(kept + at, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = activated(v[e], ACT);
        }
        if constexpr (DROP) v = dropped(v, philox((uint64_t)at >> 2, drop.k0, drop.k1), drop);
        store4(y + at, v + ahead);
    }
    // what the result is added to, where it is read ahead
    __device__ __forceinline__ floatx4 ask(int64_t row, int64_t col) const {
        return quads && residual ? load4(residual + row * cols + col) : floatx4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void operator()(floatx4 v, int64_t row, int64_t col, floatx4 ahead) const {
        const int64_t at = row * cols + col;
        v *= scale;
        if (quads) {
            if (bias) v += load4(bias + col);
            if (kept) store4(kept + at, v);
            if (act != BPT_ACT_NONE) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = activated(v[e], act);
            }
            if (drop.thr) v = dropped(v, philox((uint64_t)at >> 2, drop.k0, drop.k1), drop);
            if (residual) v += ahead;
            store4(y + at, v);
            return;
        }
        uintx4 words{0u, 0u, 0u, 0u};
        if (drop.thr) words = drop_words((uint64_t)at, drop);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (col + e >= cols) break;
            float x = v[e];
            if (bias) x += Elem<T>::ld(bias + col + e);
            if (kept) Elem<T>::st(kept + at + e, x);
            x = activated(x, act);
            if (drop.thr) x = words[e] >= drop.thr ? x * drop.inv : 0.f;
            if (residual) x += Elem<T>::ld(residual + at + e);
            Elem<T>::st(y + at + e, x);
        }
    }
};

// ---- products on tiles ----------------------------------------------------------------------------------------------------------
// out[q][p] = sum over r of B(q, r) A(p, r), P columns next to each other in memory.  The three products of a layer:
//   forward  A = weight (p, r) by rows,       B = x (q, r) by rows
//   dx       A = weight, (r, p) in memory,    B = g by rows
//   dweight  A = x, (r, p) in memory,         B = g, (r, q) in memory
// A workgroup owns a tile of BP x BQ; the reduction goes through LDS RB bytes a row at a time, two buffers: while one is multiplied, the other's
// 16-byte loads are on their way straight into LDS.  Bound by matrix instructions where the reduction is long (bfloat16 65535 x 4096 -> 1024: 457 to 600 us
// a product, 915 to 1200 TFLOP/s), by the epilogue's memory and vector instructions where it is short.  Fragments are 16 rows x 16 bytes a lane: one
// 16x16x32 product in bfloat16, four 16x16x4 in float32, whose reduction indices (4 g + j for lane group g and product j) only have to agree
// between the operands.  A is the matrix instructions' first operand, so a lane ends with four neighbouring columns of a row.
// An operand by rows lies in LDS as rows of RB / 16 chunks, shifted by row (rows_shift): the sixteen rows that a fragment reads at one chunk
// spread over the banks.  One that has the reduction outside lies as rows of the tile's elements; float32 fragments are read word by word, bfloat16
// ones by transposing loads (lane i of sixteen gives the address of 4 columns of row i / 4 and gets column i of four rows), and chunks are
// shifted by row so that the four lane groups meet different banks.
// The last step of a ragged reduction loads what lies behind it too (up to the matrix' end, where the descriptor ends), and its fragments are made zero there.
// Rows that do not start on 4 bytes, and float32's last step, go through registers, where what lies outside is made zero.
template <typename T, int RB> constexpr int step() { return RB / (int)sizeof(T); }     // the reduction's share of one buffer

// (sixteen-byte reads go to LDS sixteen lanes at a time, of lanes 0 .. 31 those of rows 0 - 3 and 12 - 15 of one chunk with rows 4 - 11 of the next)
template <int RB> __device__ __forceinline__ int rows_shift(int row) { return RB == 128 ? row & 7 : ((row >> 2 ^ row >> 3) & 1) << 1 | (row >> 3 & 1); }
template <typename T, int TB> __device__ __forceinline__ int cols_shift(int r) {
    constexpr int CHUNKS = TB * (int)sizeof(T) / 16;
    if constexpr (sizeof(T) == 4) return ((r >> 2 & 3) << 2) & (CHUNKS - 1);
    return (((r & 3) | (r >> 3 & 1) << 2) << 1) & (CHUNKS - 1);
}

// VE elements of a line from p on, of which `n` exist (the others: zero)
template <typename T> __device__ __forceinline__ uintx4 load_upto(const T *p, int64_t n) {
    typedef typename Raw<T>::type raw;
    if (n >= ve<T>()) return *reinterpret_cast<const typename Raw<T>::vec *>(p);
    uint64_t half[2] = {0, 0};
#pragma unroll 1
    for (int e = 0; e < (int)n; ++e) {
        const int bit = e * 8 * (int)sizeof(T);
        const uint64_t x = (uint64_t) reinterpret_cast<const raw *>(p)[e] << (bit & 63);
        half[0] |= bit < 64 ? x : 0;
        half[1] |= bit < 64 ? 0 : x;
    }
    return uintx4{(uint32_t)half[0], (uint32_t)(half[0] >> 32), (uint32_t)half[1], (uint32_t)(half[1] >> 32)};
}

// Sixteen bytes a lane from memory straight to LDS, lane l's to byte 16 l from `to` on (of the wavefront): a buffer descriptor of the matrix from a uniform start to its end,
// behind which nothing is read, and an offset a lane, so nothing is added per lane and load.  In assembly, because the compiler takes every transposing read of LDS for one
// that may read what is still on its way and waits for it; the waits are written where they belong (wait_and_meet), and no register is written.
__device__ __forceinline__ uint32_t lds_place(const char *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)p; }
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x);
}
__device__ __forceinline__ uintx4 memory_from(uint64_t at, uint64_t end) {      // (both uniform)
    const uint64_t bytes = end - at;
    uint32_t high = (uint32_t)(bytes >> 32);
    asm volatile("" : "+s"(high));                                 // (a minimum of 64 bits would be a vector comparison)
    uintx4 d{(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, high ? 0xffffffffu : (uint32_t)bytes, 0x00027000u};
    asm volatile("s_nop 4" : "+s"(d));                             // (a scalar register that a vector instruction wrote may be read by a load five states later)
    return d;
}
__device__ __forceinline__ void load_to_lds(uintx4 from, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(from) : "memory", "m0");
}

// one operand's way from memory to LDS
template <typename T, int TB, int RB, int WAVES, bool COLS> struct Stage {
    static constexpr int N = TB * RB / 16 / (WAVES * WAVE), VE = ve<T>(), CHUNKS = COLS ? TB * (int)sizeof(T) / 16 : RB / 16;
    const T *base;               // of this tile's first row (column) and the first step
    uint64_t from, end;          // its address, that behind the matrix, and from step to step
    int64_t apart;
    int64_t ld, stride;          // elements of a row in memory; from step to step
    int left, reduce;            // rows (columns) from base on; the reduction's length from base on
    uint32_t off[N];             // bytes from base, of a lane's vectors where they are whole

    static __device__ __forceinline__ int slot(int i) { return (i * WAVES + (int)(threadIdx.x >> 6)) * WAVE + (int)(threadIdx.x & 63); }
    static __device__ __forceinline__ int line(int i) { return slot(i) / CHUNKS; }
    static __device__ __forceinline__ int first(int i) {           // first element of the vector within its line
        const int l = line(i);
        return ((slot(i) % CHUNKS) ^ (COLS ? cols_shift<T, TB>(l) : rows_shift<RB>(l))) * VE;
    }
    // (a stage starts at step s of the reduction and tile row / column t)
    __device__ __forceinline__ Stage(const T *p, int64_t ld_, int64_t n, int64_t reduce_, int64_t t, int64_t s) : ld(ld_) {
        const int64_t r0 = s * step<T, RB>();
        base = COLS ? p + r0 * ld + t : p + t * ld + r0;
        from = uniform((uint64_t)base);
        end = uniform((uint64_t)(p + ((COLS ? reduce_ : n) - 1) * ld + (COLS ? n : reduce_)));
        stride = COLS ? ld * step<T, RB>() : step<T, RB>();
        apart = (int64_t)uniform((uint64_t)(stride * (int64_t)sizeof(T)));
        left = (int)(n - t < TB ? n - t : TB);
        reduce = (int)(reduce_ - r0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            // (past the end: the last row, the vector with a row's last element; nothing of them is stored)
            const int l = COLS ? line(i) : min(line(i), left - 1), f = COLS ? min(first(i), (left - 1) / VE * VE) : first(i);
            off[i] = (uint32_t)((l * ld + f) * (int64_t)sizeof(T));
        }
    }
    __device__ __forceinline__ void direct(int s, const char *lds) const {
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_place(lds) + (threadIdx.x >> 6) * (WAVE * 16));
        const uintx4 here = memory_from(from + s * apart, end);
#pragma unroll
        for (int i = 0; i < N; ++i) load_to_lds(here, off[i], to + i * (WAVES * WAVE * 16));
    }
    __device__ __forceinline__ void load(int s, uintx4 (&v)[N]) const {
        const T *const at = base + s * stride;
        const int rest = reduce - s * step<T, RB>();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int l = line(i), f = first(i), lines = COLS ? rest : left, cols = COLS ? left : rest;
            v[i] = l < lines ? load_upto(at + l * ld + f, cols - f) : uintx4{0u, 0u, 0u, 0u};
        }
    }
    __device__ __forceinline__ void store(const uintx4 (&v)[N], char *lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i) *reinterpret_cast<uintx4 *>(lds + slot(i) * 16) = v[i];
    }
};

// the 16 bytes that a lane has of fragment rows from .. from + 15 at bytes 64 part .. of a buffer's rows
template <typename T, int TB, int RB, bool COLS> __device__ __forceinline__ uintx4 fragment(const char *lds, int from, int part) {
    const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    if constexpr (!COLS) {
        return *reinterpret_cast<const uintx4 *>(lds + (from + c) * RB + ((part * 4 + g) ^ rows_shift<RB>(c)) * 16);
    } else if constexpr (sizeof(T) == 4) {
        uintx4 v;
        const int r = part * 16 + 4 * g, col = from + c;
        const char *const p = lds + r * (TB * 4) + (((col >> 2) ^ cols_shift<T, TB>(r)) << 4) + (col & 3) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t *>(p + j * (TB * 4));
        return v;
    } else {
        uintx4 v;
        const int col = from + (c & 3) * 4;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int r = part * 32 + 8 * g + 4 * t + (c >> 2);
            const char *const p = lds + r * (TB * 2) + (((col >> 3) ^ cols_shift<T, TB>(r)) << 4) + (col & 7) * 2;
            const shortx4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)const_cast<char *>(p));
            const uintx2v w = __builtin_bit_cast(uintx2v, x);
            v[2 * t] = w[0];
            v[2 * t + 1] = w[1];
        }
        return v;
    }
}
template <typename T> __device__ __forceinline__ floatx4 multiply(uintx4 a, uintx4 b, floatx4 c) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
}

__device__ __forceinline__ void wait_for_lds() { __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 3 << 14); }
// Eight float32, times 2^23, as three bfloat16 each, exactly: the upper 16 bits, those of what is left, and what is left then (8 + 8 + 8 digits).  bfloat16's lowest number is 2^-133, and
// digits of thirds below it would be lost: 2^23 takes the last digit of float32's lowest, 2^-149, to 2^-126, so that every third is a normal number.  (Rounded instead of cut, the thirds
// would have either sign, and what the products leave out too; but the units round sums of either sign less well: 3 x 16744449 comes out a step off, and it takes 1 to 4 percent longer.)
constexpr float THIRDS_BY = 0x1p23f, THIRDS_BACK = 0x1p-46f;       // (of an operand; of a product of two)
__device__ __forceinline__ void thirds(uintx4 a, uintx4 b, uintx4 (&out)[3]) {
    uint32_t x[8], y[8], z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = __float_as_uint(__uint_as_float(e < 4 ? a[e & 3] : b[e & 3]) * THIRDS_BY);
        y[e] = __float_as_uint(__uint_as_float(x[e]) - __uint_as_float(x[e] & 0xffff0000u));
        z[e] = __float_as_uint(__uint_as_float(y[e]) - __uint_as_float(y[e] & 0xffff0000u));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        out[0][e] = __builtin_amdgcn_perm(x[2 * e + 1], x[2 * e], 0x07060302u);
        out[1][e] = __builtin_amdgcn_perm(y[2 * e + 1], y[2 * e], 0x07060302u);
        out[2][e] = __builtin_amdgcn_perm(z[2 * e + 1], z[2 * e], 0x07060302u);
    }
}

// Waits until at most N of this wavefront's loads are on their way and all that it has asked of LDS is there, then for the workgroup.
template <int N> __device__ __forceinline__ void wait_and_meet() {
    issue_loads_first();
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    wait_for_lds();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue_loads_first();
}
// The order of what has been written since the last fence: reads of LDS spread evenly between matrix products.
template <int READS, int PRODUCTS> __device__ __forceinline__ void in_turn() {
    constexpr int EACH = PRODUCTS / READS > 0 ? PRODUCTS / READS : 1;
#pragma unroll
    for (int i = 0; i < READS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    }
}

struct Product {
    int64_t P, Q, R;             // columns, rows, reduction
    int64_t lda, ldb;
    int tiles_p, tiles, splits;  // tiles of a row of them, of the result; shares of the reduction
    int steps, per_split;        // steps of the reduction, of a share
};

// The tiles' shapes: columns, rows, wavefronts over either, bytes of a row and step, buffers, workgroups a compute unit.
template <int BP_, int BQ_, int GP_, int GQ_, int PER_CU_> struct Shape {
    static constexpr int BP = BP_, BQ = BQ_, GP = GP_, GQ = GQ_, RB = 128, STAGES = 2, WAVES = GP * GQ, THREADS = WAVES * WAVE;
    static constexpr int PER_SIMD = (PER_CU_ * WAVES + 3) / 4;     // wavefronts that share a vector unit's registers
};

// The sums leave through LDS, so that a row of the tile is written (and bias, residual read) as one run of memory.
// part: null, or (splits, Q, P) sums of the shares, which k_linear_finish adds up
template <typename T, typename S, bool ACOLS, bool BCOLS, bool DIRECT, bool THIRDS>
__global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void k_linear_tiles(const T *__restrict__ a, const T *__restrict__ b, Product m, Epilogue<T> out, float *__restrict__ part) {
    constexpr int BP = S::BP, BQ = S::BQ, RB = S::RB, STAGES = S::STAGES;
    constexpr int WP = BP / S::GP, WQ = BQ / S::GQ, FP = WP / 16, FQ = WQ / 16;        // a wavefront's part of the tile, in fragments
    constexpr int BUFFER = (BP + BQ) * RB;
    constexpr int PASSES = BP * BQ * 4 <= STAGES * BUFFER ? 1 : 2, JS = FQ / PASSES, ROWS = S::GQ * 16 * JS;      // of sums that LDS takes at a time, fragments and rows
    static_assert(ROWS * BP * 4 <= STAGES * BUFFER, "");
    __shared__ __attribute__((aligned(16))) char lds[STAGES * BUFFER];
    const int id = xcd_contiguous_block(), split = id / m.tiles, tile = id - split * m.tiles;
    const int64_t q0 = (int64_t)(tile / m.tiles_p) * BQ, p0 = (int64_t)(tile % m.tiles_p) * BP;
    const int s0 = split * m.per_split, n = min(m.per_split, m.steps - s0);
    typedef Stage<T, BP, RB, S::WAVES, ACOLS> StageA;
    typedef Stage<T, BQ, RB, S::WAVES, BCOLS> StageB;
    const StageA sa(a, m.lda, m.P, m.R, p0, s0);
    const StageB sb(b, m.ldb, m.Q, m.R, q0, s0);
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, wp = w % S::GP * WP, wq = w / S::GP * WQ;
    floatx4 acc[FP][FQ];
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
        for (int j = 0; j < FQ; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    uintx4 fa[2][FP], fb[2][FQ];
    auto read = [&](int into, const char *at, int half) {
#pragma unroll
        for (int i = 0; i < FP; ++i) fa[into][i] = fragment<T, BP, RB, ACOLS>(at, wp + 16 * i, half);
#pragma unroll
        for (int j = 0; j < FQ; ++j) fb[into][j] = fragment<T, BQ, RB, BCOLS>(at + BP * RB, wq + 16 * j, half);
    };
    auto products = [&](int of) {
#pragma unroll
        for (int j = 0; j < FQ; ++j)
#pragma unroll
            for (int i = 0; i < FP; ++i) acc[i][j] = multiply<T>(fa[of][i], fb[of][j], acc[i][j]);
    };
    // float32 by the bfloat16 units: six of the nine products of thirds.  The second third is below 2^-7 of an operand and the last below 2^-15, so what is left out is below
    // 2^-21 (1 + 2^-9) of |a| |b| (of random digits 2^-24.6 on the mean), always towards zero
    auto products_of_thirds = [&](const char *at) {
        uintx4 ta[FP][3], raw[2][2];
        auto read_b = [&](int j) {
#pragma unroll
            for (int half = 0; half < 2; ++half) raw[j & 1][half] = fragment<T, BQ, RB, BCOLS>(at + BP * RB, wq + 16 * j, half);
        };
#pragma unroll
        for (int i = 0; i < FP; ++i) thirds(fragment<T, BP, RB, ACOLS>(at, wp + 16 * i, 0), fragment<T, BP, RB, ACOLS>(at, wp + 16 * i, 1), ta[i]);
        read_b(0);
#pragma unroll
        for (int j = 0; j < FQ; ++j) {
            issue_loads_first();                                   // (a fragment ahead, not all of them: they would not fit)
            if (j + 1 < FQ) read_b(j + 1);
            uintx4 tb[3];
            thirds(raw[j & 1][0], raw[j & 1][1], tb);
            constexpr int OF[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
#pragma unroll
            for (int t = 0; t < 6; ++t)
#pragma unroll
                for (int i = 0; i < FP; ++i) acc[i][j] = multiply<bf16_t>(ta[i][OF[t][0]], tb[OF[t][1]], acc[i][j]);
        }
    };
    int s = 0;
    if constexpr (DIRECT) {
        constexpr int LOADS = StageA::N + StageB::N;
        const int whole = min(n, sa.reduce / step<T, RB>());       // (of n steps; the one behind them is ragged)
        auto ask = [&](int t) {
            char *const at = lds + (t & 1) * BUFFER;
            sa.direct(t, at);
            sb.direct(t, at + BP * RB);
        };
        if constexpr (THIRDS) {
            if (whole > 0) ask(0);
            for (; s < whole; ++s) {
                wait_and_meet<0>();                                // (step s is there, step s - 1 has been read by all)
                if (s + 1 < whole) ask(s + 1);
                products_of_thirds(lds + (s & 1) * BUFFER);
            }
        } else {
            // Half a step's products run while the other half's fragments, or the next step's first, are read:
            //   products of (s, 0), reads of (s, 1)  |  step s + 1 is there, step s has been read by all: step s + 2 is asked for  |  products of (s, 1), reads of (s + 1, 0)
            constexpr int READS = FP * (ACOLS ? (sizeof(T) == 4 ? 4 : 2) : 1) + FQ * (BCOLS ? (sizeof(T) == 4 ? 4 : 2) : 1), PRODUCTS = FP * FQ * (sizeof(T) == 4 ? 4 : 1);
            if (n > 0) {
                ask(0);
                if (n > 1) {
                    ask(1);
                    wait_and_meet<LOADS>();
                } else {
                    wait_and_meet<0>();
                }
                read(0, lds, 0);
            }
            for (; s < whole; ++s) {
                wait_for_lds();                                    // (before the next reads, not behind the first of them)
                issue_loads_first();
                read(1, lds + (s & 1) * BUFFER, 1);
                products(0);
                in_turn<READS, PRODUCTS>();
                wait_and_meet<0>();
                if (s + 2 < n) ask(s + 2);
                issue_loads_first();
                read(0, lds + (~s & 1) * BUFFER, 0);               // (behind the last step: what the buffer held, for nobody)
                products(1);
                in_turn<READS, PRODUCTS>();
                issue_loads_first();
            }
            if (s < n) {
                read(1, lds + (s & 1) * BUFFER, 1);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int there = sa.reduce - s * step<T, RB>() - (half * 4 + (lane >> 4)) * ve<T>();      // of the lane's elements
                    static_assert(sizeof(T) == 2, "");
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const uint32_t mask = there >= 2 * d + 2 ? 0xffffffffu : there == 2 * d + 1 ? 0xffffu : 0u;
#pragma unroll
                        for (int i = 0; i < FP; ++i) fa[half][i][d] &= mask;
#pragma unroll
                        for (int j = 0; j < FQ; ++j) fb[half][j][d] &= mask;
                    }
                    products(half);
                }
                s = n;
            }
        }
    }
    // Steps first .. n - 1 through registers.
    auto through_registers = [&](int first, bool in_thirds) {
        if (first >= n) return;
        uintx4 va[StageA::N], vb[StageB::N];
        sa.load(first, va);
        sb.load(first, vb);
        __syncthreads();
        for (int t = first; t < n; ++t) {
            char *const at = lds + (t & 1) * BUFFER;               // (what it held was read before the last barrier)
            sa.store(va, at);
            sb.store(vb, at + BP * RB);
            __syncthreads();
            if (t + 1 < n) {
                sa.load(t + 1, va);
                sb.load(t + 1, vb);
            }
            if (THIRDS && in_thirds) {
                products_of_thirds(at);
            } else {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    read(0, at, half);
                    products(0);
                }
            }
        }
    };
    if constexpr (!THIRDS) {
        if constexpr (!DIRECT) through_registers(s, false);
    } else {
        // Thirds of an infinity are infinity and NaN, and numbers of 2^105 and above, or sums of 2^82, leave float32's range times 2^23 or 2^46: a tile with a sum that is not finite is
        // formed again by the float32 instructions.
        through_registers(s, true);
        float odd = 0.f;
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) odd = fmaf(acc[i][j][e], 0.f, odd);
        const bool again = __syncthreads_or(!(odd == 0.f));
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
            for (int j = 0; j < FQ; ++j) acc[i][j] = again ? floatx4{0.f, 0.f, 0.f, 0.f} : acc[i][j] * THIRDS_BACK;
        if (again) through_registers(0, false);
    }
    // the tile, or half of every wavefront's rows at a time, as rows of BP floats, quad i of row r at i ^ r: sixteen rows' quads of a fragment spread over the banks
    constexpr int QUADS = BP / 4, TURNS = ROWS * QUADS / S::THREADS, U = 4;
    floatx4 *const sums = reinterpret_cast<floatx4 *>(lds);
    const int quad = threadIdx.x % QUADS;
    const int64_t p = p0 + quad * 4;
    const int left = (int)(m.Q - q0 < BQ ? m.Q - q0 : BQ);
    const bool mine = p < m.P;
    const floatx4 none{0.f, 0.f, 0.f, 0.f}, bias = mine && out.quads && out.bias && !part ? load4(out.bias + p) : none;
    auto put = [&](auto pass) {
#pragma unroll
        for (int j = 0; j < JS; ++j)
#pragma unroll
            for (int i = 0; i < FP; ++i) {
                const int r = w / S::GP * (16 * JS) + 16 * j + (lane & 15), to = (wp + 16 * i) / 4 + (lane >> 4);
                sums[r * QUADS + (to ^ (r & (QUADS - 1)))] = acc[i][pass() * JS + j];
            }
    };
#pragma unroll 1
    for (int pass = 0; pass < PASSES; ++pass) {
        auto line = [&](int u) { return u * (S::THREADS / QUADS) + (int)threadIdx.x / QUADS; };                         // of the sums,
        auto row = [&](int u) { return line(u) / (16 * JS) * WQ + pass * (16 * JS) + line(u) % (16 * JS); };            // of the tile
        auto sum = [&](int u) { return sums[line(u) * QUADS + (quad ^ (line(u) & (QUADS - 1)))]; };
        auto at = [&](int u) { return (q0 + row(u)) * m.P + p; };
        floatx4 ahead[U];
        auto ask = [&](int u0) {
#pragma unroll
            for (int u = 0; u < U; ++u) ahead[u] = row(u0 + u) < left ? load4(out.residual + at(u0 + u)) : none;
        };
        const bool added = mine && out.quads && out.residual && !part;
#pragma unroll
        for (int u = 0; u < U; ++u) ahead[u] = none;
        if (added) ask(0);
        __syncthreads();
        if (PASSES == 1 || pass == 0) put(std::integral_constant<int, 0>{});
        else put(std::integral_constant<int, PASSES - 1>{});
        __syncthreads();
        if (!mine) continue;
        if (part) {
            float *const to = part + (int64_t)split * m.Q * m.P;
#pragma unroll U
            for (int u = 0; u < TURNS; ++u) {
                if (row(u) >= left) continue;
                const floatx4 v = sum(u);
                if ((m.P & 3) == 0) {
                    store4(to + at(u), v);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (p + e < m.P) to[at(u) + e] = v[e];
                }
            }
            continue;
        }
        constexpr bool FORWARD = !ACOLS && !BCOLS;
        if (!out.quads || (FORWARD && out.act == BPT_ACT_NONE && out.kept)) {
#pragma unroll 1
            for (int u = 0; u < TURNS; ++u)
                if (row(u) < left) out(sum(u), q0 + row(u), p, FORWARD ? out.ask(q0 + row(u), p) : none);
            continue;
        }
        // a loop for each activation, with dropout or without (asked for each four columns, that took 7 us of 50 of a product of 33598 x 300 -> 600 without any)
        auto leave = [&](auto act, auto drop) {
#pragma unroll 1
            for (int u0 = 0; u0 < TURNS; u0 += U) {
                floatx4 now[U];
#pragma unroll
                for (int u = 0; u < U; ++u) now[u] = ahead[u];
                if (added && u0 + U < TURNS) ask(u0 + U);
                issue_loads_first();
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (row(u0 + u) < left) out.template quad<act(), drop()>(sum(u0 + u), at(u0 + u), bias, now[u]);
            }
        };
        using std::integral_constant;
        auto with_drop = [&](auto act) {
            if (out.drop.thr) leave(act, integral_constant<bool, true>{});
            else leave(act, integral_constant<bool, false>{});
        };
        if constexpr (!FORWARD) {                                  // (the backward's products: nothing follows them)
            leave(integral_constant<int, BPT_ACT_NONE>{}, integral_constant<bool, false>{});
        } else {
            if (out.act == BPT_ACT_RELU) with_drop(integral_constant<int, BPT_ACT_RELU>{});
            else if (out.act == BPT_ACT_GELU) with_drop(integral_constant<int, BPT_ACT_GELU>{});
            else with_drop(integral_constant<int, BPT_ACT_NONE>{});
        }
    }
}

// the shares' sums in their order, and what follows the product
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_linear_finish(const float *__restrict__ part, int splits, int64_t rows, int64_t cols, Epilogue<T> out) {
    const int64_t quads = (cols + 3) / 4, i = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
    if (i >= rows * quads) return;
    const int64_t row = i / quads, col = (i - row * quads) * 4, n = rows * cols;
    const float *const p = part + row * cols + col;
    floatx4 v{0.f, 0.f, 0.f, 0.f};
    if ((cols & 3) == 0) {
        int s = 0;
        for (; s + 4 <= splits; s += 4) {
            floatx4 t[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) t[u] = load4(p + (s + u) * n);
#pragma unroll
            for (int u = 0; u < 4; ++u) v += t[u];
        }
        for (; s < splits; ++s) v += load4(p + s * n);
    } else {
        for (int s = 0; s < splits; ++s) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < cols) v[e] += p[s * n + e];
        }
    }
    out(v, row, col, out.ask(row, col));
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------------
// Forward of up to 16 NQ rows: bound by the latency of reading the weight once (1 x 512 -> 2048 float32 4.2 us, 48 x 512 -> 512 bfloat16 4.9 us; a launch of nothing takes 2).
// A workgroup has 16 columns and all rows, its wavefronts share the reduction and meet in LDS; fragments come straight from memory, sixteen lanes' rows of 64 bytes each.
constexpr int FEW_WAVES = 8;
template <typename T, bool WHOLE> __device__ __forceinline__ uintx4 few_load(const T *row, int64_t k, int64_t R) {
    if constexpr (WHOLE) {
        if (k < R) return *reinterpret_cast<const uintx4 *>(row + k);
        return uintx4{0u, 0u, 0u, 0u};
    }
    return k < R ? load_upto(row + k, R - k) : uintx4{0u, 0u, 0u, 0u};
}
template <typename T, int NQ, bool WHOLE>
__global__ __launch_bounds__(FEW_WAVES *WAVE) void k_linear_few(const T *__restrict__ w, const T *__restrict__ x, int64_t P, int64_t Q, int64_t R, Epilogue<T> out) {
    constexpr int K = 4 * ve<T>();                                 // the reduction's share of a fragment
    __shared__ floatx4 meet[FEW_WAVES][NQ][WAVE];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int64_t p0 = (int64_t)blockIdx.x * 16, p = p0 + c;
    const T *const wr = w + (p < P ? p : P - 1) * R;
    const T *xr[NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) xr[j] = x + (16 * j + c < Q ? 16 * j + c : Q - 1) * R;
    floatx4 acc[NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
    constexpr int U = NQ == 1 ? 4 : NQ == 2 ? 4 : 2;
    for (int64_t k0 = (int64_t)wave * K; k0 < R; k0 += (int64_t)FEW_WAVES * K * U) {
        uintx4 a[U], b[U][NQ];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = k0 + (int64_t)u * FEW_WAVES * K + g * ve<T>();
            a[u] = few_load<T, WHOLE>(wr, k, R);
#pragma unroll
            for (int j = 0; j < NQ; ++j) b[u][j] = few_load<T, WHOLE>(xr[j], k, R);
        }
        issue_loads_first();
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < NQ; ++j) acc[j] = multiply<T>(a[u], b[u][j], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < NQ; ++j) meet[wave][j][lane] = acc[j];
    __syncthreads();
    for (int j = wave; j < NQ; j += FEW_WAVES) {
        floatx4 v = meet[0][j][lane];
#pragma unroll
        for (int i = 1; i < FEW_WAVES; ++i) v += meet[i][j][lane];
        const int64_t q = 16 * j + c, col = p0 + 4 * g;
        if (q < Q && col < P) out(v, q, col, out.ask(q, col));
    }
}

// ---- the gradient before the products ------------------------------------------------------------------------------------------
// g = dy keep act'(a), keep 0 or 1, and the sums of its columns: bound by memory, dy and a read and g written once (65535 x 1024 bfloat16 with dropout 75 to 85 us, 3.4 TB/s:
// the generator's products are as long; 33598 x 600 gelu 38 us, 3.2 TB/s; 16383 x 2048 float32 relu 69 us, 5.8 TB/s, y still in the last cache).  What dropout divides by is
// left to the products and the sums, in 32 bits: without an activation, and with relu, g is dy where it is not 0, and nothing is rounded.  A workgroup has 64 lanes' columns
// (four each) and every parts-th four rows; its wavefronts meet in LDS, the workgroups in k_linear_sums, in a fixed order.
template <typename T>
__global__ __launch_bounds__(BLOCK) void k_linear_grad(const T *dy, const T *__restrict__ kept, int kept_is_result, T *g, float *__restrict__ part, int64_t rows,
                                                       int64_t cols, int act, Drop drop, bool quads) {
    __shared__ floatx4 meet[WAVES_PER_BLOCK][WAVE];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t col = ((int64_t)blockIdx.x * WAVE + lane) * 4;
    constexpr int U = 4;
    floatx4 sum{0.f, 0.f, 0.f, 0.f};
    const int64_t stride = (int64_t)gridDim.y * WAVES_PER_BLOCK;
    for (int64_t row = (int64_t)blockIdx.y * WAVES_PER_BLOCK + wave; row < rows; row += stride * U) {
        floatx4 v[U], a[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = row + u * stride, at = r * cols + col;
            v[u] = a[u] = floatx4{0.f, 0.f, 0.f, 0.f};
            if (r >= rows || col >= cols) continue;
            if (quads) {
                v[u] = load4(dy + at);
                if (act != BPT_ACT_NONE) a[u] = load4(kept + at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < cols) {
                        v[u][e] = Elem<T>::ld(dy + at + e);
                        if (act != BPT_ACT_NONE) a[u][e] = Elem<T>::ld(kept + at + e);
                    }
            }
        }
        issue_loads_first();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = row + u * stride, at = r * cols + col;
            if (r >= rows || col >= cols) continue;
            if (drop.thr && !kept_is_result) v[u] = dropped(v[u], drop_words((uint64_t)at, drop), drop);      // (what was dropped is 0 in the result; drop.inv is 1)
            if (act != BPT_ACT_NONE) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[u][e] = activated_back(v[u][e], a[u][e], act);
            }
            if (quads) {
                if (g) store4(g + at, v[u]);
                sum += v[u];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < cols) {
                        if (g) Elem<T>::st(g + at + e, v[u][e]);
                        sum[e] += v[u][e];
                    }
            }
        }
    }
    if (!part) return;
    meet[wave][lane] = sum;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 1; i < WAVES_PER_BLOCK; ++i) sum += meet[i][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < cols) part[(int64_t)blockIdx.y * cols + col + e] = sum[e];
}
// 16 columns a workgroup, sixteen lanes a column take parts p, p + 16, ...; the sixteen are added in their order
template <typename T> __global__ __launch_bounds__(BLOCK) void k_linear_sums(const float *__restrict__ part, int parts, T *__restrict__ out, int64_t cols, float scale) {
    __shared__ float meet[16][17];
    const int c = threadIdx.x & 15, k = threadIdx.x >> 4;
    for (int64_t first = (int64_t)blockIdx.x * 16; first < cols; first += (int64_t)gridDim.x * 16) {
        const int64_t at = first + c;
        float v = 0.f;
        if (at < cols) {
            int p = k;
            for (; p + 15 * 16 < parts; p += 16 * 16) {
                float t[16];
#pragma unroll
                for (int u = 0; u < 16; ++u) t[u] = part[(int64_t)(p + u * 16) * cols + at];
#pragma unroll
                for (int u = 0; u < 16; ++u) v += t[u];
            }
            for (; p < parts; p += 16) v += part[(int64_t)p * cols + at];
        }
        __syncthreads();                                           // (the turn before has been read)
        meet[k][c] = v;
        __syncthreads();
        if (k != 0 || at >= cols) continue;
        v = meet[0][c];
#pragma unroll
        for (int i = 1; i < 16; ++i) v += meet[i][c];
        Elem<T>::st(out + at, v * scale);
    }
}

// ---- dropout -----------------------------------------------------------------------------------------------------------------------
// y = residual + dropout(x): bound by memory, the words are formed while the loads are on their way.  A lane has four vectors of 16 bytes.  65535 x 1024 bfloat16 57 us each way
// (4.7 TB/s, as a large copy); 16383 x 512 float32 11 and 17 us, the latter with a residual (6 TB/s: much of it is in the last cache).
template <typename T, bool AL>
__global__ __launch_bounds__(BLOCK) void k_dropout(const T *x, const T *residual, T *y, int64_t n, Drop drop) {
    constexpr int VE = ve<T>(), U = 4;
    typedef typename Raw<T>::vec loose;
    const int64_t first = ((int64_t)blockIdx.x * U * BLOCK + threadIdx.x) * VE;
    auto fetch = [](const T *p) -> uintx4 {
        if constexpr (AL) return *reinterpret_cast<const uintx4 *>(p);
        return *reinterpret_cast<const loose *>(p);
    };
    auto wide = [](uintx4 v, int h) {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(floatx4, v);
        return floatx4{__uint_as_float(v[2 * h] << 16), __uint_as_float(v[2 * h] & 0xffff0000u), __uint_as_float(v[2 * h + 1] << 16),
                       __uint_as_float(v[2 * h + 1] & 0xffff0000u)};
    };
    uintx4 vx[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = first + (int64_t)u * BLOCK * VE;
        if (at + VE > n) continue;
        vx[u] = fetch(x + at);
        if (residual) vr[u] = fetch(residual + at);
    }
    issue_loads_first();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t at = first + (int64_t)u * BLOCK * VE;
        if (at + VE <= n) {
            uintx4 o;
#pragma unroll
            for (int h = 0; h < VE / 4; ++h) {
                floatx4 v = dropped(wide(vx[u], h), philox((uint64_t)(at >> 2) + h, drop.k0, drop.k1), drop);
                if (residual) v += wide(vr[u], h);
                if constexpr (sizeof(T) == 4) {
                    o = __builtin_bit_cast(uintx4, v);
                } else {
                    o[2 * h] = pack_bf16(v[0], v[1]);
                    o[2 * h + 1] = pack_bf16(v[2], v[3]);
                }
            }
            if constexpr (AL) *reinterpret_cast<uintx4 *>(y + at) = o;
            else *reinterpret_cast<loose *>(y + at) = o;
        } else if (at < n) {
#pragma unroll
            for (int h = 0; h < VE / 4; ++h) {
                const uintx4 words = philox((uint64_t)(at >> 2) + h, drop.k0, drop.k1);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t i = at + 4 * h + e;
                    if (i >= n) continue;
                    float v = words[e] >= drop.thr ? Elem<T>::ld(x + i) * drop.inv : 0.f;
                    if (residual) v += Elem<T>::ld(residual + i);
                    Elem<T>::st(y + i, v);
                }
            }
        }
    }
}

// ---- launchers -------------------------------------------------------------------------------------------------------------------
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline bool on(std::initializer_list<const void *> ps, uintptr_t bytes) {
    for (const void *p : ps)
        if ((uintptr_t)p % bytes) return false;
    return true;
}

// Which tiles, and into how many shares the reduction goes.  256 x 256: one workgroup a compute unit, LDS and caches are asked for least, but nothing runs beside its
// start and end: where a round of the chip is filled (or, by shares, a long reduction fills it) and those are a small part.  128 x 128: two a unit, where they fill the chip, by
// shares too if the reduction is longer than what their sums cost on the way through memory.  64 x 64: where the larger ones would leave units idle.
// us, by 256 | 128 | 64, bfloat16 (forward of rows x inner -> outer): 65535 x 4096 -> 1024 457 | 582 | 931, 8192 x 4096 -> 4096 223 | 285 | 565, 16383 x 512 -> 2048 45 | 50 | 66,
// 16383 x 2048 -> 512 55 | 37 | 51, 2000 x 512 -> 2048 20 | 10 | 11, 1023 x 512 -> 512 19 | 9.2 | 8.8; dweight (shares) of 65535 x 4096 -> 1024 475 | 577 | 1226, of 16383 x 512 -> 2048
// 52 | 45 | 71; float32 4096 x 4096 -> 4096 657 | 729 | 986, 16383 x 512 -> 2048 187 | 197 | 272, 1023 x 512 -> 512 77 | 23 | 14.
// Two or three shares on 128 x 128 | one on 64 x 64, bfloat16: 4096 x 1024 -> 1024 27 | 17, 2500 x 2048 -> 1024 26 | 22, 2500 x 4096 -> 1024 35 | 41; float32: 3000 x 512 -> 1024 38 | 29,
// 4096 x 1024 -> 1024 59 | 67, 2048 x 1024 -> 2048 61 | 71.  320 tiles of 128 x 128 | 64 x 64: dx of 2500 x 2048 -> 1024 20 | 24, float32 89 | 89.
// Shares of 4 | 8 | 16 steps at least on 64 x 64, bfloat16: 65 x 512 -> 512 9.6 | 5.9 | 5.8, 256 x 1024 -> 1024 8.7 | 8.8 | 7.9, 1023 x 512 -> 512 8.9 | 5.8 | 5.8, 256 x 2048 -> 512 8.6 | 8.8 | 10.1;
// float32: 65 x 512 -> 512 10.6 | 12.1 | 15.8, 127 x 768 -> 768 10.9 | 12.7 | 22, 256 x 1024 -> 1024 14.9 | 13.9 | 19, dweight of 256 x 512 -> 2048 15.4 | 10.4 | 10.4.
typedef Shape<256, 256, 4, 2, 1> Huge;
typedef Shape<128, 128, 2, 2, 2> Large;
typedef Shape<64, 64, 2, 2, 4> Small;
enum Tiles { HUGE, LARGE, SMALL };
struct Choice {
    Tiles tiles;
    int splits;
};
template <typename T> inline Choice choose(int64_t P, int64_t Q, int64_t R) {
    auto count = [&](int64_t b) { return ceil_div(P, b) * ceil_div(Q, b); };
    const int64_t steps = ceil_div(R, 128 / (int64_t)sizeof(T)), huge = count(256), large = count(128), small = count(64);
    if (R >= 1024 && huge >= 192 && 4 * huge >= 3 * 256 * ceil_div(huge, 256)) return Choice{HUGE, 1};
    if (steps >= 512 && huge >= 32 && huge < 192) return Choice{HUGE, (int)(256 / huge)};
    constexpr bool LOW = sizeof(T) == 2;
    if (large >= (LOW ? 272 : 384)) return Choice{LARGE, 1};
    if (small >= 512 && R <= (LOW ? 2048 : 512)) return Choice{SMALL, 1};
    const int64_t large_splits = std::max<int64_t>(1, std::min<int64_t>(steps / 8, 512 / large)), share = small >= 64 ? 8 : 4;
    const int64_t small_splits = LOW && steps <= 16 ? 1 : std::max<int64_t>(1, std::min<int64_t>(steps / share, 512 / small));
    if (large * large_splits >= 384) return Choice{LARGE, (int)large_splits};
    return Choice{SMALL, (int)small_splits};
}
// f(shape) of a choice
template <typename T, typename F> inline auto with_shape(Tiles tiles, F &&f) {
    if (tiles == HUGE) return f(Huge{});
    return tiles == LARGE ? f(Large{}) : f(Small{});
}
template <typename T> inline Product product(int64_t P, int64_t Q, int64_t R, int64_t lda, int64_t ldb, const Choice &ch) {
    return with_shape<T>(ch.tiles, [&](auto shape) {
        typedef decltype(shape) S;
        Product m{P, Q, R, lda, ldb, 0, 0, 0, 0, 0};
        m.tiles_p = (int)ceil_div(P, S::BP);
        m.tiles = (int)(m.tiles_p * ceil_div(Q, S::BQ));
        m.steps = (int)ceil_div(R, step<T, S::RB>());
        m.per_split = (int)ceil_div(m.steps, ch.splits);
        m.splits = (int)ceil_div(m.steps, m.per_split);
        return m;
    });
}
template <typename T> inline int64_t product_workspace(int64_t P, int64_t Q, int64_t R) {
    const Product m = product<T>(P, Q, R, 0, 0, choose<T>(P, Q, R));
    return m.splits > 1 ? (int64_t)m.splits * P * Q * 4 : 0;
}

// out's rows and columns are the product's
template <typename T, bool AC, bool BC>
int run_product(const T *a, const T *b, int64_t P, int64_t Q, int64_t R, int64_t lda, int64_t ldb, const Epilogue<T> &out, void *ws, hipStream_t s) {
    const Choice ch = choose<T>(P, Q, R);
    const Product m = product<T>(P, Q, R, lda, ldb, ch);
    float *const part = m.splits > 1 ? (float *)ws : nullptr;
    // Straight to LDS: rows that start on 4 bytes, as loads of several words do (33598 x 300 -> 600 bfloat16, through registers / straight: dx 64 / 30 us, dweight 79 / 29), and hold
    // a vector at least; a lane's offsets into a step count 32 bits (256 rows of 2^21 elements).
    const bool direct = on({a, b}, 4) && lda * sizeof(T) % 4 == 0 && ldb * sizeof(T) % 4 == 0 && std::min(lda, ldb) >= ve<T>() && std::max(lda, ldb) <= (int64_t)1 << 21;
    const dim3 grid((unsigned)(m.tiles * (int64_t)m.splits));
    const int st = with_shape<T>(ch.tiles, [&](auto shape) {
        typedef decltype(shape) S;
        if (direct) hipLaunchKernelGGL((k_linear_tiles<T, S, AC, BC, true, sizeof(T) == 4>), grid, dim3(S::THREADS), 0, s, a, b, m, out, part);
        else hipLaunchKernelGGL((k_linear_tiles<T, S, AC, BC, false, sizeof(T) == 4>), grid, dim3(S::THREADS), 0, s, a, b, m, out, part);
        return launch_status();
    });
    if (st != BPT_OK || !part) return st;
    hipLaunchKernelGGL((k_linear_finish<T>), dim3((unsigned)ceil_div(Q * ceil_div(P, 4), BLOCK)), dim3(BLOCK), 0, s, part, m.splits, Q, P, out);
    return launch_status();
}
template <typename T> inline Epilogue<T> plain_epilogue(T *y, int64_t cols, double scale) {
    return Epilogue<T>{nullptr, nullptr, y, nullptr, cols, (float)scale, BPT_ACT_NONE, make_drop(0.0, 0), cols % 4 == 0 && on({y}, 4 * sizeof(T))};
}

// Whether the kernel of few rows takes a forward: every workgroup of it reads all of x, 128 KB at most where it has more than a fragment's rows.  us, few rows | tiles, bfloat16:
// 16 x 512 -> 512 4.9 | 7.2, 16 x 4096 -> 4096 9.8 | 10.4, 64 x 512 -> 512 4.8 | 6.8, 64 x 1024 -> 4096 7.2 | 8.8, 32 x 2048 -> 512 7.6 | 6.8, 64 x 2048 -> 512 11.5 | 8.3, 64 x 4096 -> 4096
// 21 | 12.5; float32 16 x 4096 -> 4096 19 | 32, 64 x 512 -> 512 8.0 | 10.5, 32 x 1024 -> 4096 9.2 | 12.9, 64 x 1024 -> 1024 12.5 | 10.6, 32 x 2048 -> 512 14 | 10.8, 64 x 4096 -> 4096 43 | 34.
// (A launch counts its threads in 32 bits: of more columns the tiles have fewer.)
inline bool few_rows(int64_t rows, int64_t inner, int64_t outer, int64_t size) {
    return (rows <= 16 || (rows <= 64 && rows * inner * size <= (int64_t)1 << 17)) && outer <= (int64_t)1 << 26;
}
template <typename T>
int run_forward(const void *x_, const void *w_, const void *b_, const void *r_, void *y_, void *kept_, void *ws, int64_t rows, int64_t inner, int64_t outer, int act,
                Drop drop, hipStream_t s) {
    const T *x = (const T *)x_, *w = (const T *)w_;
    const Epilogue<T> out{(const T *)b_, (const T *)r_, (T *)y_, (T *)kept_, outer, 1.f, act, drop, outer % 4 == 0 && on({b_, r_, y_, kept_}, 4 * sizeof(T))};
    if (few_rows(rows, inner, outer, sizeof(T))) {
        const bool whole = inner % ve<T>() == 0 && on({x, w}, 16);
        const dim3 grid((unsigned)ceil_div(outer, 16)), block(FEW_WAVES * WAVE);
#define LAUNCH(NQ) \
    if (whole) hipLaunchKernelGGL((k_linear_few<T, NQ, true>), grid, block, 0, s, w, x, outer, rows, inner, out); \
    else hipLaunchKernelGGL((k_linear_few<T, NQ, false>), grid, block, 0, s, w, x, outer, rows, inner, out)
        if (rows <= 16) { LAUNCH(1); }
        else if (rows <= 32) { LAUNCH(2); }
        else { LAUNCH(4); }
#undef LAUNCH
        return launch_status();
    }
    return run_product<T, false, false>(w, x, outer, rows, inner, inner, inner, out, ws, s);
}

// workgroups that share the rows of one strip of 256 columns
inline int grad_parts(int64_t rows, int64_t cols) {
    const int64_t strips = ceil_div(cols, 4 * WAVE);
    return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, 4 * WAVES_PER_BLOCK), ceil_div(2048, strips)));
}
template <typename T>
int run_grad(const void *dy_, const void *kept_, int result, void *g_, void *db_, void *ws, int64_t rows, int64_t cols, int act, Drop drop, hipStream_t s) {
    const int parts = grad_parts(rows, cols);
    const bool quads = cols % 4 == 0 && on({dy_, act != BPT_ACT_NONE ? kept_ : nullptr, g_}, 4 * sizeof(T));
    float *const part = db_ ? (float *)ws : nullptr;
    const float inv = drop.inv;
    drop.inv = 1.f;
    if (rows > 0)
        hipLaunchKernelGGL((k_linear_grad<T>), dim3((unsigned)ceil_div(cols, 4 * WAVE), parts), dim3(BLOCK), 0, s, (const T *)dy_, (const T *)kept_, result, (T *)g_, part,
                           rows, cols, act, drop, quads);
    const int st = launch_status();
    if (st != BPT_OK || !db_) return st;
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(cols, 16), (int64_t)1 << 20);      // (a launch counts its threads in 32 bits)
    hipLaunchKernelGGL((k_linear_sums<T>), dim3(blocks), dim3(BLOCK), 0, s, part, rows > 0 ? parts : 0, (T *)db_, cols, inv);
    return launch_status();
}

template <typename T> int run_dropout(const void *x, const void *r, void *y, int64_t n, Drop drop, hipStream_t s) {
    if (n > (((int64_t)1 << 32) - BLOCK) * 4 * ve<T>()) return BPT_ERR_SIZE;      // (a launch counts its threads in 32 bits)
    const dim3 grid((unsigned)ceil_div(n, (int64_t)BLOCK * 4 * ve<T>()));
    if (on({x, r, y}, 16)) hipLaunchKernelGGL((k_dropout<T, true>), grid, dim3(BLOCK), 0, s, (const T *)x, (const T *)r, (T *)y, n, drop);
    else hipLaunchKernelGGL((k_dropout<T, false>), grid, dim3(BLOCK), 0, s, (const T *)x, (const T *)r, (T *)y, n, drop);
    return launch_status();
}

inline bool is_type(int dtype) { return dtype == BPT_F32 || dtype == BPT_BF16; }
inline bool is_share(double p) { return p >= 0.0 && p < 1.0; }
// (grids count tiles, quads and rows in 31 bits)
inline bool is_size(int64_t rows, int64_t inner, int64_t outer) {
    const int64_t most = (int64_t)1 << 28;
    if (rows < 0 || inner < 1 || outer < 0 || rows > most || inner > most || outer > most) return false;
    const double cells = 1.0 * ((int64_t)1 << 38);
    return (double)rows * outer <= cells && (double)rows * inner <= cells && (double)inner * outer <= cells;
}

}  // namespace

extern "C" {

#define FOR_TYPE(call) (dtype == BPT_F32 ? call<float> : call<bf16_t>)

int64_t bpt_linear_forward_workspace_bytes(int64_t rows, int64_t inner, int64_t outer, int dtype) {
    if (!is_type(dtype) || !is_size(rows, inner, outer)) return -1;
    if (few_rows(rows, inner, outer, dtype == BPT_F32 ? 4 : 2) || outer == 0) return 0;
    return FOR_TYPE(product_workspace)(outer, rows, inner);
}

int bpt_linear_forward(const void *x, const void *weight, const void *bias, const void *residual, void *y, void *kept, void *workspace, int64_t workspace_bytes,
                       int64_t rows, int64_t inner, int64_t outer, int act, double dropout_p, uint64_t seed, int dtype, void *stream) {
    if (!is_type(dtype)) return BPT_ERR_DTYPE;
    if (!is_size(rows, inner, outer) || !is_share(dropout_p)) return BPT_ERR_SIZE;
    if (act < BPT_ACT_NONE || act > BPT_ACT_GELU) return BPT_ERR_UNSUPPORTED;
    if (rows == 0 || outer == 0) return BPT_OK;
    if (!x || !weight || !y) return BPT_ERR_NULL;
    const int64_t need = bpt_linear_forward_workspace_bytes(rows, inner, outer, dtype);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return BPT_ERR_WORKSPACE;
    return FOR_TYPE(run_forward)(x, weight, bias, residual, y, kept, workspace, rows, inner, outer, act, make_drop(dropout_p, seed), (hipStream_t)stream);
}

int64_t bpt_linear_grad_workspace_bytes(int64_t rows, int64_t outer, int dtype) {
    if (!is_type(dtype) || !is_size(rows, 1, outer)) return -1;
    return outer == 0 ? 0 : (int64_t)grad_parts(rows, outer) * outer * 4;
}

int bpt_linear_grad(const void *dy, const void *kept, int kept_is_result, void *g, void *dbias, void *workspace, int64_t workspace_bytes, int64_t rows, int64_t outer,
                    int act, double dropout_p, uint64_t seed, int dtype, void *stream) {
    if (!is_type(dtype)) return BPT_ERR_DTYPE;
    if (!is_size(rows, 1, outer) || !is_share(dropout_p)) return BPT_ERR_SIZE;
    if (act < BPT_ACT_NONE || act > BPT_ACT_GELU || (kept_is_result && act != BPT_ACT_RELU)) return BPT_ERR_UNSUPPORTED;
    if (outer == 0 || (!g && !dbias) || (rows == 0 && !dbias)) return BPT_OK;
    if (rows > 0 && (!dy || (act != BPT_ACT_NONE && !kept))) return BPT_ERR_NULL;
    if (dbias && (!workspace || workspace_bytes < bpt_linear_grad_workspace_bytes(rows, outer, dtype) || !aligned16(workspace))) return BPT_ERR_WORKSPACE;
    return FOR_TYPE(run_grad)(dy, kept, kept_is_result, g, dbias, workspace, rows, outer, act, make_drop(dropout_p, seed), (hipStream_t)stream);
}

int64_t bpt_linear_input_grad_workspace_bytes(int64_t rows, int64_t inner, int64_t outer, int dtype) {
    if (!is_type(dtype) || !is_size(rows, inner, outer) || outer < 1) return -1;
    return rows == 0 ? 0 : FOR_TYPE(product_workspace)(inner, rows, outer);
}

int bpt_linear_input_grad(const void *g, const void *weight, void *dx, void *workspace, int64_t workspace_bytes, int64_t rows, int64_t inner, int64_t outer,
                          double scale, int dtype, void *stream) {
    if (!is_type(dtype)) return BPT_ERR_DTYPE;
    if (!is_size(rows, inner, outer) || outer < 1) return BPT_ERR_SIZE;
    if (rows == 0) return BPT_OK;
    if (!g || !weight || !dx) return BPT_ERR_NULL;
    const int64_t need = bpt_linear_input_grad_workspace_bytes(rows, inner, outer, dtype);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return BPT_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == BPT_F32)
        return run_product<float, true, false>((const float *)weight, (const float *)g, inner, rows, outer, inner, outer, plain_epilogue((float *)dx, inner, scale), workspace, s);
    return run_product<bf16_t, true, false>((const bf16_t *)weight, (const bf16_t *)g, inner, rows, outer, inner, outer, plain_epilogue((bf16_t *)dx, inner, scale), workspace, s);
}

int64_t bpt_linear_weight_grad_workspace_bytes(int64_t rows, int64_t inner, int64_t outer, int dtype) {
    if (!is_type(dtype) || !is_size(rows, inner, outer) || rows < 1) return -1;
    return outer == 0 ? 0 : FOR_TYPE(product_workspace)(inner, outer, rows);
}

int bpt_linear_weight_grad(const void *g, const void *x, void *dweight, void *workspace, int64_t workspace_bytes, int64_t rows, int64_t inner, int64_t outer,
                           double scale, int dtype, void *stream) {
    if (!is_type(dtype)) return BPT_ERR_DTYPE;
    if (!is_size(rows, inner, outer) || rows < 1) return BPT_ERR_SIZE;
    if (outer == 0) return BPT_OK;
    if (!g || !x || !dweight) return BPT_ERR_NULL;
    const int64_t need = bpt_linear_weight_grad_workspace_bytes(rows, inner, outer, dtype);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return BPT_ERR_WORKSPACE;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == BPT_F32)
        return run_product<float, true, true>((const float *)x, (const float *)g, inner, outer, rows, inner, outer, plain_epilogue((float *)dweight, inner, scale), workspace, s);
    return run_product<bf16_t, true, true>((const bf16_t *)x, (const bf16_t *)g, inner, outer, rows, inner, outer, plain_epilogue((bf16_t *)dweight, inner, scale), workspace, s);
}

int bpt_dropout(const void *x, const void *residual, void *y, int64_t n, double dropout_p, uint64_t seed, int dtype, void *stream) {
    if (!is_type(dtype)) return BPT_ERR_DTYPE;
    if (n < 0 || n > (int64_t)1 << 40 || !is_share(dropout_p)) return BPT_ERR_SIZE;
    if (n == 0) return BPT_OK;
    if (!x || !y) return BPT_ERR_NULL;
    return FOR_TYPE(run_dropout)(x, residual, y, n, make_drop(dropout_p, seed), (hipStream_t)stream);
}

#undef FOR_TYPE

}  // extern "C"
