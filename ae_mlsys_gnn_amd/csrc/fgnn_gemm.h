// Products of dense matrices on the matrix instructions, the core of the dense operators:
//     D[m][n] = sum_k Q(m, k) P(n, k)          rows m, columns n (contiguous in D), reduction k
// Either operand comes with its reduction contiguous ("C": element (i, k) at p[i ld + k]) or strided ("S": at p[k ld + i]), so that a forward
// product (C, C), the gradient of its input (P strided) and of its weights (both strided) read the matrices as they lie in memory.
//
// P is the first operand of the instructions: a lane ends up with four consecutive n of one m, the four lanes of a row with 16.  Results of 16 bits want eight
// (16 bytes) a lane: then the tiles of P are interleaved in pairs (instruction row r of tile t is n = 32 (t / 2) + 8 (r / 4) + 4 (t % 2) + r % 4).  Either way
// one store instruction writes 64 bytes of each of 16 rows, as do reads of the residual (with 16 columns a lane, in four stores of 16 bytes each 64
// apart, the L2 saw four times the requests: 169,343 x 128 -> 256 fp32 with gelu and residual 226 us).
//
// Element kinds: 16-bit values (exact products, summed in 32 bits), 8-bit integers (summed in integers, over the parts of a cut reduction too: exact), 8-bit
// floats, and fp32.  fp32 operands are cut into three parts of 8 significant bits (truncated, so that the three are exact), and the six products that reach above
// 2^-24 of the result are summed in 32 bits: the matrix unit does 16 of them in the time of one fp32 product.
#pragma once
#include <algorithm>
#include <type_traits>
#include "fgnn_elem.h"

typedef float gm_f4 __attribute__((ext_vector_type(4)));
typedef int gm_i4 __attribute__((ext_vector_type(4)));
typedef short gm_s4 __attribute__((ext_vector_type(4)));
typedef __bf16 gm_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 gm_h8 __attribute__((ext_vector_type(8)));

enum { GM_NONE = 0, GM_RELU = 1, GM_GELU = 2, GM_SILU = 3, GM_LEAKY = 4 };

// The normal distribution's function P(z) and exp(-z^2 / 2), which its slope needs too.  P(-|z|) = t (c1 + .. + c5 t^4) exp(-z^2 / 2) with t = 1 / (1 + p |z|)
// (Hastings' approximation, Abramowitz and Stegun 26.2.17: off by 7.5e-8 at the most); one exponential and one reciprocal where the library's erff takes some
// fifty instructions, which no other workgroup's products hide in the epilogue (169,343 x 128 -> 256 fp32 with gelu and residual 275 / 224 us).
__device__ __forceinline__ float gm_normal(float z, float &bell)
{
    const float t = __builtin_amdgcn_rcpf(fmaf(0.2316419f, fabsf(z), 1.f));
    bell = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
    const float c = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.330274429f, -1.821255978f), 1.781477937f), -0.356563782f), 0.319381530f);
    const float below = c * (0.39894228f * bell);
    return z > 0.f ? 1.f - below : z == z ? below : z;
}
__device__ __forceinline__ float gm_logistic(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }

template <int W>
__device__ __forceinline__ void gm_act(float (&z)[W], int act, float slope)
{
    float bell;
    switch (act) {
    case GM_RELU:
#pragma unroll
        for (int i = 0; i < W; ++i) z[i] = z[i] > 0.f ? z[i] : z[i] == z[i] ? 0.f : z[i];
        break;
    case GM_GELU:
#pragma unroll
        for (int i = 0; i < W; ++i) z[i] *= gm_normal(z[i], bell);
        break;
    case GM_SILU:
#pragma unroll
        for (int i = 0; i < W; ++i) z[i] *= gm_logistic(z[i]);
        break;
    case GM_LEAKY:
#pragma unroll
        for (int i = 0; i < W; ++i) z[i] = z[i] > 0.f ? z[i] : slope * z[i];
        break;
    }
}
// Far out gelu and silu are straight: what is outside +-128 has the slope that is there, 0 or 1 in 32 bits.  (z comes rounded to the rows' type: of fp16 an infinity
// may stand for an argument that the forward pass had as a finite number.)  A NaN stays one.
__device__ __forceinline__ float gm_within(float z) { return z > 128.f ? 128.f : z < -128.f ? -128.f : z; }
// g times the slope at z
template <int W>
__device__ __forceinline__ void gm_act_slope(float (&g)[W], const float (&z)[W], int act, float slope)
{
    switch (act) {
    case GM_RELU:
#pragma unroll
        for (int i = 0; i < W; ++i) g[i] = z[i] > 0.f ? g[i] : 0.f;
        break;
    case GM_GELU:
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float bell;
            const float u = gm_within(z[i]), p = gm_normal(u, bell);
            g[i] *= fmaf(u, 0.39894228f * bell, p);
        }
        break;
    case GM_SILU:
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float u = gm_within(z[i]), p = gm_logistic(u);
            g[i] *= fmaf(p * u, 1.f - p, p);
        }
        break;
    case GM_LEAKY:
#pragma unroll
        for (int i = 0; i < W; ++i) g[i] *= z[i] > 0.f ? 1.f : slope;
        break;
    }
}

// What becomes of the sums: y = act(z) + residual, z = acc sx[m] sw[n] + bias[n], in type E.
struct GemmEpi {
    int64_t m; int n;
    const float *sx, *sw;                   // NULL: 1
    const void *bias; int btype;
    const void *res; int64_t ldr;
    int act; float slope;
    void *z, *y;                            // contiguous [m, n]; z NULL: not wanted
};

// W consecutive elements of a row, the first `count` of them where fewer are left.
template <typename E, int W, typename U>
__device__ __forceinline__ void gm_load(U (&v)[W], const E *p, int count)
{
    constexpr int V = fe_width<E> < W ? fe_width<E> : W;
    typedef E vec __attribute__((ext_vector_type(V), aligned(sizeof(E))));
    if (count >= W) {
#pragma unroll
        for (int j = 0; j < W / V; ++j) {
            const vec u = *reinterpret_cast<const vec *>(p + j * V);
#pragma unroll
            for (int i = 0; i < V; ++i) v[j * V + i] = (U)u[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = i < count ? (U)p[i] : (U)0;
    }
}
template <typename E, int W, typename U>
__device__ __forceinline__ void gm_store(const U (&v)[W], E *p, int count)
{
    constexpr int V = fe_width<E> < W ? fe_width<E> : W;
    typedef E vec __attribute__((ext_vector_type(V), aligned(sizeof(E))));
    if (count >= W) {
#pragma unroll
        for (int j = 0; j < W / V; ++j) {
            vec u;
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] = (E)v[j * V + i];
            *reinterpret_cast<vec *>(p + j * V) = u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) if (i < count) p[i] = (E)v[i];
    }
}

// The W columns n .. n + W - 1 that a lane works on: what does not depend on the row is read once.
template <int W> struct GemmCols { float bias[W], sw[W]; };
template <int W>
__device__ __forceinline__ void gm_columns(const GemmEpi &e, int n, GemmCols<W> &c)
{
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const int j = n + i < e.n ? n + i : e.n - 1;
        c.bias[i] = e.bias ? fe_load(e.bias, j, e.btype) : 0.f;
        c.sw[i] = e.sw ? e.sw[j] : 1.f;
    }
}
template <typename E, int W> struct GemmVec { typedef E type __attribute__((ext_vector_type(W), aligned(sizeof(E)))); };
// The residual's W values at (m, n) where all of them exist (anything else: read one by one later), asked for ahead of their use.
template <typename E, int W>
__device__ __forceinline__ typename GemmVec<E, W>::type gm_ahead(const GemmEpi &e, int64_t m, int n)
{
    typename GemmVec<E, W>::type u = {};
    if (e.res && e.n >= W) {
        const bool there = m < e.m && n + W <= e.n;
        u = *reinterpret_cast<const typename GemmVec<E, W>::type *>((const E *)e.res + (there ? m * e.ldr + n : 0));
    }
    return u;
}
template <typename E, int W>
__device__ __forceinline__ void gm_finish(const GemmEpi &e, const GemmCols<W> &c, const typename GemmVec<E, W>::type &ahead, int64_t m, int n, float (&v)[W])
{
    const int count = e.n - n;
    if (m >= e.m || count <= 0) return;
    const int64_t at = m * e.n + n;
    if (e.sx) {
        const float s = e.sx[m];
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] *= s * c.sw[i];
    }
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += c.bias[i];
    if (e.z) gm_store<E, W>(v, (E *)e.z + at, count);
    if (e.act) gm_act(v, e.act, e.slope);
    if (e.res) {
        float r[W];
#pragma unroll
        for (int i = 0; i < W; ++i) r[i] = (float)ahead[i];
        if (count < W) gm_load<E, W>(r, (const E *)e.res + m * e.ldr + n, count);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] += r[i];
    }
    gm_store<E, W>(v, (E *)e.y + at, count);
}

struct GemmP {
    int64_t m, k;
    int n;
    const void *q, *p; int64_t ldq, ldp;
    int tiles_m, tiles_n, splits;
    int lower;                              // only tiles on and below the diagonal: D is symmetric, and the epilogue writes the rest
    int64_t slabs;                          // slabs of the reduction a split takes
    void *part;                             // [splits][m][n] where splits > 1, in the type of the sums: fp32, or int32 of 8-bit integers
    int64_t rows_q, rows_p;                 // rows that the operands have (more than D has where a strided one is padded to whole chunks)
    int64_t batch_q, batch_p, plane_q, plane_p;                                // bytes between the batch's matrices, and between planes
    GemmEpi epi;
};

// Workgroup w runs on XCD w % 8: every XCD gets a run of neighbouring tiles, eight rows of tiles high, so that its L2 holds what they share.
__device__ __forceinline__ void gm_tile(const GemmP &p, int &tm, int &tn, int &split)
{
    const int total = (int)gridDim.x, b = (int)blockIdx.x, xcd = b % FGNN_NUM_XCD, q = total / FGNN_NUM_XCD, r = total % FGNN_NUM_XCD;
    int t = xcd * q + min(xcd, r) + b / FGNN_NUM_XCD;
    const int tiles = p.lower ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n;
    split = t / tiles;
    t -= split * tiles;
    if (p.lower) {
        tm = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
        while (tm * (tm + 1) / 2 > t) --tm;
        while ((tm + 1) * (tm + 2) / 2 <= t) ++tm;
        tn = t - tm * (tm + 1) / 2;
        return;
    }
    constexpr int HIGH = 8;
    const int band = t / (HIGH * p.tiles_n), first = band * HIGH, high = min(HIGH, p.tiles_m - first);
    t -= band * HIGH * p.tiles_n;
    tm = first + t % high;
    tn = t / high;
}

// ------------------------------------------------------------------------------------------------ element kinds
template <int KIND> struct GemmKind {       // 16-bit values
    static constexpr int planes = 1, slab = 64, size = 2, chunk = 8, words = 4;
    typedef gm_f4 acc;
};
template <> struct GemmKind<FGNN_F32> {     // slab: reduction elements a tile; chunk: elements a thread loads at a time, as `words` registers
    static constexpr int planes = 3, slab = 32, size = 4, chunk = 8, words = 8;
    typedef gm_f4 acc;
};
template <> struct GemmKind<FGNN_I8> {
    static constexpr int planes = 1, slab = 128, size = 1, chunk = 16, words = 4;
    typedef gm_i4 acc;
};
template <> struct GemmKind<FGNN_E4M3> {    // wait in LDS as fp16, which holds them exactly: see gm_widen
    static constexpr int planes = 1, slab = 64, size = 1, chunk = 16, words = 4;
    typedef gm_f4 acc;
};

// LDS tile of an operand with `rows` rows (of D's rows or columns), one plane of a slab.  C: [rows][row bytes], 64 bytes a row for fp32's parts and 128
// else; S: [slab][rows] 16-bit values.  16-byte chunks of a row are exchanged so that the lanes of one LDS pass meet different banks.
template <int KIND> constexpr int gm_row_bytes = GemmKind<KIND>::slab *(KIND == FGNN_I8 ? 1 : 2);
template <int RB, bool PAIRS>
__device__ __forceinline__ int gm_at_c(int row, int chunk)
{
    const int f = RB == 64 ? (row >> 1) & 3 : PAIRS ? (row & 3) | ((row >> 3) & 1) << 2 : row & 7;
    return row * RB + ((chunk ^ f) << 4);
}
template <int ROWS, bool PAIRS>
__device__ __forceinline__ int gm_at_s(int k, int chunk)
{
    const int f = PAIRS ? (k & 3) << 2 : (k & 3) << 1;
    return k * (ROWS * 2) + ((chunk ^ f) << 4);
}

// Operand registers of 16 rows (tile t; the tiles of a 64-row block may be interleaved in pairs) and one instruction's reduction.
template <int RB, int ROWS, bool S, bool PAIRS>
__device__ __forceinline__ gm_i4 gm_operand(const char *tile, int t, int step, int lane)
{
    static_assert(!(PAIRS && RB == 64) && ROWS >= 128, "the exchanges of chunks stay within a row");
    const int r = lane & 15, g = lane >> 4;
    if constexpr (!S) {
        const int row = PAIRS ? 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3) : 16 * t + r;
        return *reinterpret_cast<const gm_i4 *>(tile + gm_at_c<RB, PAIRS>(row, 4 * step + g));
    } else {
        // the transposing read: 16 lanes give four rows of 16 values (four a lane) and get a column of four each
        const int i = PAIRS ? 32 * (t >> 1) + 8 * (r & 3) + 4 * (t & 1) : 16 * t + 4 * (r & 3);
        const int k = 32 * step + 8 * g + (r >> 2);
        typedef __attribute__((address_space(3))) gm_s4 *lds_p;
        const char *a = tile + gm_at_s<ROWS, PAIRS>(k, i >> 3) + ((i >> 2) & 1) * 8;
        const gm_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)a), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(a + 4 * ROWS * 2));
        typedef short s8 __attribute__((ext_vector_type(8)));
        const s8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return *reinterpret_cast<const gm_i4 *>(&v);
    }
}

template <int KIND>
__device__ __forceinline__ typename GemmKind<KIND>::acc gm_mfma(gm_i4 a, gm_i4 b, typename GemmKind<KIND>::acc c)
{
    if constexpr (KIND == FGNN_I8) return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
    else if constexpr (KIND == FGNN_F16 || KIND == FGNN_E4M3) return __builtin_amdgcn_mfma_f32_16x16x32_f16(*(gm_h8 *)&a, *(gm_h8 *)&b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(gm_b8 *)&a, *(gm_b8 *)&b, c, 0, 0, 0);
}
// One slab: a wave's 64 columns (block wp of P's tile) by 16 TQ rows (16-row tiles from tq0 on of Q's).
template <int KIND, int BM, int BN, bool QS, bool PS, bool PAIRS, int TQ>
__device__ __forceinline__ void gm_slab(const char *lq, const char *lp, int wp, int tq0, int lane, typename GemmKind<KIND>::acc (&acc)[TQ][4])
{
    constexpr int PLQ = BM * GemmKind<KIND>::slab * 2, PLP = BN * GemmKind<KIND>::slab * 2;      // bytes a plane (where there are several)
    if constexpr (KIND == FGNN_F32) {
        gm_i4 a[4][3];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < 3; ++h) a[t][h] = gm_operand<gm_row_bytes<KIND>, BN, PS, PAIRS>(lp + h * PLP, 4 * wp + t, 0, lane);
#pragma unroll
        for (int q = 0; q < TQ; ++q) {
            gm_i4 b[3];
#pragma unroll
            for (int h = 0; h < 3; ++h) b[h] = gm_operand<gm_row_bytes<KIND>, BM, QS, false>(lq + h * PLQ, tq0 + q, 0, lane);
            // the small products first
#pragma unroll
            for (int s = 2; s >= 0; --s)
#pragma unroll
                for (int h = 0; h <= s; ++h)
#pragma unroll
                    for (int t = 0; t < 4; ++t) acc[q][t] = gm_mfma<FGNN_BF16>(a[t][s - h], b[h], acc[q][t]);
        }
    } else {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            gm_i4 a[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) a[t] = gm_operand<gm_row_bytes<KIND>, BN, PS, PAIRS>(lp, 4 * wp + t, s, lane);
#pragma unroll
            for (int q = 0; q < TQ; ++q) {
                const gm_i4 b = gm_operand<gm_row_bytes<KIND>, BM, QS, false>(lq, tq0 + q, s, lane);
#pragma unroll
                for (int t = 0; t < 4; ++t) acc[q][t] = gm_mfma<KIND>(a[t], b, acc[q][t]);
            }
        }
    }
}

// What becomes of W sums a lane, as the kernels take it: LinearEpi for linear maps.  ROWS: rows whose reads are asked for together.
template <typename E>
struct LinearEpi {
    static constexpr int W = fe_width<E>, ROWS = 4;
    GemmEpi e;
    typedef GemmCols<W> Cols;
    typedef typename GemmVec<E, W>::type Ahead;
    __device__ __forceinline__ void columns(int n, Cols &c) const { gm_columns(e, n, c); }
    __device__ __forceinline__ Ahead ahead(int64_t, int64_t m, int n) const { return gm_ahead<E, W>(e, m, n); }
    __device__ __forceinline__ void finish(const Cols &c, const Ahead &a, int64_t, int64_t m, int n, float (&v)[W]) const { gm_finish<E, W>(e, c, a, m, n, v); }
};

// A wave's results: 16 TQ rows from m0 on, 64 columns from n0 on.
template <int TQ, typename F, typename A>
__device__ __forceinline__ void gm_results(const GemmP &p, const F &f, int64_t batch, int split, int64_t m0, int n0, int lane, const A (&acc)[TQ][4])
{
    constexpr int W = F::W, J = 16 / W, ROWS = F::ROWS < TQ ? F::ROWS : TQ;
    const int r = lane & 15, g = lane >> 4;
    auto sums = [&]<typename U>(int i, int j, U (&v)[W]) {
#pragma unroll
        for (int k = 0; k < W; ++k) v[k] = (U)acc[i][j * (W / 4) + k / 4][k % 4];
    };
    auto column = [&](int j) { return n0 + 4 * W * j + W * g; };
    if (p.splits > 1) {
        typedef std::remove_reference_t<decltype(acc[0][0][0] + acc[0][0][0])> S;           // float, or int of 8-bit integers
#pragma unroll
        for (int i = 0; i < TQ; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int64_t m = m0 + 16 * i + r;
                S v[W];
                sums(i, j, v);
                if (m < p.m && column(j) < p.n) gm_store<S, W>(v, (S *)p.part + ((batch * p.splits + split) * p.m + m) * p.n + column(j), p.n - column(j));
            }
        return;
    }
    typename F::Cols cols[J];
#pragma unroll
    for (int j = 0; j < J; ++j) f.columns(column(j), cols[j]);
    // a row's parts one after the other: lines of the caches that are written whole leave them whole
#pragma unroll
    for (int i0 = 0; i0 < TQ; i0 += ROWS) {
        typename F::Ahead a[ROWS][J];
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) a[i][j] = f.ahead(batch, m0 + 16 * (i0 + i) + r, column(j));
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) {
                float v[W];
                sums(i0 + i, j, v);
                f.finish(cols[j], a[i][j], batch, m0 + 16 * (i0 + i) + r, column(j), v);
            }
    }
}

// ------------------------------------------------------------------------------------------------ operands of any alignment, through registers
// `words` registers of CH elements, the first `valid` of them from memory and zeros after them.
template <int KIND>
__device__ __forceinline__ void gm_fetch(uint32_t (&w)[GemmKind<KIND>::words], const char *p, int valid)
{
    constexpr int CH = GemmKind<KIND>::chunk, SIZE = GemmKind<KIND>::size, W = GemmKind<KIND>::words;
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(1)));
    if (valid >= CH) {
#pragma unroll
        for (int j = 0; j < W / 4; ++j) {
            const u4 u = reinterpret_cast<const u4 *>(p)[j];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * j + i] = u[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i < valid) {
                if constexpr (SIZE == 4) w[i] = ((const uint32_t *)p)[i];
                else if constexpr (SIZE == 2) w[i / 2] |= (uint32_t)((const uint16_t *)p)[i] << (16 * (i & 1));
                else w[i / 4] |= (uint32_t)((const uint8_t *)p)[i] << (8 * (i & 3));
            }
    }
}

// Eight fp32 values as three parts of eight significant bits that add up to them exactly.
__device__ __forceinline__ void gm_split(const uint32_t (&w)[8], gm_i4 (&part)[3])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t p[2][3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = __uint_as_float(w[2 * j + i]);
            const uint32_t hi = w[2 * j + i] & 0xffff0000u;
            const float r1 = x - __uint_as_float(hi);           // (of an infinity or a NaN: NaN, which gm_repair sees to)
            const uint32_t mid = __float_as_uint(r1) & 0xffff0000u;
            const float r2 = r1 - __uint_as_float(mid);
            p[i][0] = hi; p[i][1] = mid; p[i][2] = __float_as_uint(r2);
        }
#pragma unroll
        for (int h = 0; h < 3; ++h) part[h][j] = (int)__builtin_amdgcn_perm(p[1][h], p[0][h], 0x07060302u);
    }
}

// Sixteen 8-bit floats as fp16, exactly.  The instructions that take 8-bit floats as they are would be twice as fast, but align the products of a sum to
// its largest with few bits below: 2^-18 of the sum of magnitudes was off for values within a factor of 32, 2^-13 over the type's whole range (2^-23 here).
__device__ __forceinline__ void gm_widen(const uint32_t (&w)[4], gm_i4 (&half)[2])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        const h2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.f, true);
        half[i / 2][2 * (i % 2)] = *(const int *)&lo;
        half[i / 2][2 * (i % 2) + 1] = *(const int *)&hi;
    }
}

template <int KIND, int ROWS, bool S, int THREADS>
struct GemmLoader {
    static constexpr int CH = GemmKind<KIND>::chunk, SLAB = GemmKind<KIND>::slab, SIZE = GemmKind<KIND>::size, W = GemmKind<KIND>::words;
    static constexpr int INNER = (S ? ROWS : SLAB) / CH, COUNT = ROWS * SLAB / CH / THREADS, STEP = THREADS / INNER;     // chunks a row, chunks and row step a thread
    static_assert(THREADS % INNER == 0 && (ROWS * SLAB / CH) % THREADS == 0, "threads share a tile evenly");
    const char *base; int64_t ld;           // ld in bytes
    int outer, inner, rows;                 // place in the tile; rows left of the operand from the tile's first on
    uint32_t w[COUNT][W];

    __device__ __forceinline__ void init(const void *p, int64_t ld_, int64_t row0, int64_t rows_, int64_t k0)
    {
        outer = (int)threadIdx.x / INNER;
        inner = (int)threadIdx.x % INNER;
        ld = ld_ * SIZE;
        rows = (int)min((int64_t)ROWS, rows_ - row0);
        base = (const char *)p + (S ? (k0 + outer) * ld + (row0 + inner * CH) * SIZE : (row0 + outer) * ld + (k0 + inner * CH) * SIZE);
    }
    // the slab that `base` stands at, of which `left` reduction elements exist; moves on
    __device__ __forceinline__ void fetch(int64_t left)
    {
        const bool whole = rows == ROWS && left >= SLAB;
#pragma unroll
        for (int c = 0; c < COUNT; ++c) {
            const int o = outer + c * STEP;
            const char *p = base + (int64_t)c * STEP * ld;
            int valid = CH;
            if (!whole) {
                if (S) valid = o < left ? rows - inner * CH : 0;
                else valid = o < rows ? (int)min((int64_t)CH, left - inner * CH) : 0;
            }
            gm_fetch<KIND>(w[c], p, valid);
        }
        base += S ? (int64_t)SLAB * ld : (int64_t)SLAB * SIZE;
    }
    template <bool PAIRS>
    __device__ __forceinline__ void store(char *tile)
    {
#pragma unroll
        for (int c = 0; c < COUNT; ++c) {
            const int o = outer + c * STEP, at = S ? gm_at_s<ROWS, PAIRS>(o, inner) : gm_at_c<gm_row_bytes<KIND>, PAIRS>(o, inner);
            if constexpr (KIND == FGNN_E4M3) {
                gm_i4 half[2];
                gm_widen(w[c], half);
#pragma unroll
                for (int h = 0; h < 2; ++h) *reinterpret_cast<gm_i4 *>(tile + gm_at_c<gm_row_bytes<KIND>, PAIRS>(o, 2 * inner + h)) = half[h];
            } else if constexpr (KIND == FGNN_F32) {
                gm_i4 part[3];
                gm_split(w[c], part);
#pragma unroll
                for (int h = 0; h < 3; ++h) *reinterpret_cast<gm_i4 *>(tile + h * (ROWS * SLAB * 2) + at) = part[h];
            } else *reinterpret_cast<gm_i4 *>(tile + at) = gm_i4{(int)w[c][0], (int)w[c][1], (int)w[c][2], (int)w[c][3]};
        }
    }
};

// Sums of fp32 parts that are no finite numbers, formed again by the fp32 instruction: an infinity times another operand's empty part is NaN, where the
// product of the whole values is an infinity.  Elements of D whose sums are finite keep them.  Straight from memory: for rows that hold infinities or NaN.
template <bool QS, bool PS, int TQ>
__device__ __forceinline__ void gm_repair(const GemmP &p, int64_t m0, int n0, int64_t k0, int64_t k1, int lane, gm_f4 (&acc)[TQ][4])
{
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int q = 0; q < TQ; ++q) {
        bool bad = false;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) bad |= !__builtin_isfinite(acc[q][t][j]);
        if (__ballot(bad) == 0) continue;
        const int64_t m = min(m0 + 16 * q + r, p.m - 1);
        gm_f4 sum[4] = {};
#pragma unroll 1
        for (int64_t k = k0; k < k1; k += 4) {
            const int64_t kk = min(k + g, k1 - 1);
            const bool in = k + g < k1;
            const float b = in ? ((const float *)p.q)[QS ? kk * p.ldq + m : m * p.ldq + kk] : 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int64_t n = min(n0 + 16 * t + r, p.n - 1);
                const float a = in ? ((const float *)p.p)[PS ? kk * p.ldp + n : n * p.ldp + kk] : 0.f;
                sum[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, sum[t], 0, 0, 0);
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) if (!__builtin_isfinite(acc[q][t][j])) acc[q][t][j] = sum[t][j];
    }
}

// 128 x 128 tiles, four waves of 64 x 64 each.  A slab waits in registers while the one before it is multiplied out of LDS; two workgroups share a compute
// unit, so that one multiplies while the other converts and stores.  fp32 8192 x 4096 -> 8192: 223 TFLOP/s, input gradient 205, weights' gradient 202, bound by the
// six products (the library's fp32 products 152, 154, 154).
template <int KIND, typename E, bool QS, bool PS>
__global__ __launch_bounds__(256, 2) void gemm_any_kernel(GemmP p)
{
    constexpr int BM = 128, BN = 128, SLAB = GemmKind<KIND>::slab, TQ = 4, W = fe_width<E>;
    constexpr bool PAIRS = W == 8;
    constexpr int BYTES = 128 * gm_row_bytes<KIND> * GemmKind<KIND>::planes;
    __shared__ __attribute__((aligned(16))) char lds[2 * BYTES];
    char *lq = lds, *lp = lds + BYTES;
    int tm, tn, split;
    gm_tile(p, tm, tn, split);
    const int lane = fg_lane(), wave = fg_wave(), wp = wave & 1, tq0 = (wave >> 1) * TQ;
    const int64_t k0 = split * p.slabs * SLAB, k1 = min(p.k, k0 + p.slabs * SLAB);
    typename GemmKind<KIND>::acc acc[TQ][4] = {};
    GemmLoader<KIND, BM, QS, 256> q;
    GemmLoader<KIND, BN, PS, 256> b;
    q.init(p.q, p.ldq, (int64_t)tm * BM, p.m, k0);
    b.init(p.p, p.ldp, (int64_t)tn * BN, p.n, k0);
    if (k0 < k1) {
        q.fetch(k1 - k0);
        b.fetch(k1 - k0);
    }
#pragma unroll 1
    for (int64_t k = k0; k < k1; k += SLAB) {
        __syncthreads();                    // the slab before has been read
        q.template store<false>(lq);
        b.template store<PAIRS>(lp);
        __syncthreads();
        if (k + SLAB < k1) {
            q.fetch(k1 - k - SLAB);
            b.fetch(k1 - k - SLAB);
        }
        gm_slab<KIND, BM, BN, QS, PS, PAIRS, TQ>(lq, lp, wp, tq0, lane, acc);
    }
    if constexpr (KIND == FGNN_F32) gm_repair<QS, PS, TQ>(p, (int64_t)tm * BM + 16 * tq0, tn * BN + 64 * wp, k0, k1, lane, acc);
    gm_results<TQ>(p, LinearEpi<E>{p.epi}, 0, split, (int64_t)tm * BM + 16 * tq0, tn * BN + 64 * wp, lane, acc);
}

// The partial sums of a reduction cut into `splits`, added up in a fixed order: four columns a thread, or a part of their sums where few columns have many.
template <typename E, typename S, int SHARE>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmP p)
{
    typedef S quad __attribute__((ext_vector_type(4)));
    __shared__ quad sums[SHARE > 1 ? 256 : 1];
    const int quads = (p.n + 3) / 4, share = (int)threadIdx.x / (256 / SHARE);
    const int64_t i = (int64_t)blockIdx.x * (256 / SHARE) + threadIdx.x % (256 / SHARE), m = i / quads;
    const int n = (int)(i - m * quads) * 4;
    S v[4] = {0, 0, 0, 0};
    if (m < p.m) {
#pragma unroll 4
        for (int s = share; s < p.splits; s += SHARE) {
            S u[4];
            gm_load<S, 4>(u, (const S *)p.part + ((int64_t)s * p.m + m) * p.n + n, p.n - n);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += u[j];
        }
    }
    if constexpr (SHARE > 1) {
        sums[threadIdx.x] = quad{v[0], v[1], v[2], v[3]};
        __syncthreads();
        if (share) return;
#pragma unroll
        for (int s = 1; s < SHARE; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += sums[s * (256 / SHARE) + threadIdx.x][j];
    }
    if (m >= p.m) return;
    GemmCols<4> cols;
    gm_columns(p.epi, n, cols);
    float z[4] = {(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
    gm_finish<E, 4>(p.epi, cols, gm_ahead<E, 4>(p.epi, m, n), m, n, z);
}

// ------------------------------------------------------------------------------------------------ aligned operands, from memory to LDS
// Operands whose rows start at 16 bytes and hold whole 16-byte chunks go from memory to LDS without passing registers.  A slab is 128 bytes of a row (whole lines
// of the caches: with 64 the L2 sees twice the requests), two instructions' reduction; LDS holds two slabs.  A wave always has a half slab's operands
// in registers and reads the next half while it multiplies, so that it meets the others once a slab, in its middle: then the next slab has arrived,
// and this one is in registers everywhere, so that its place takes the one after next.  bf16 8192 x 4096 -> 8192: 1404 TFLOP/s, input gradient 1458, weights'
// gradient 1424 (the library's products 1600, 1442, 1226), 8-bit integers 2479: bound by the matrix unit, which is busy in 69 % of the cycles (4096^3).
// PLANES = 2: both operands are hi + 2^-11 lo (`plane_q`, `plane_p` bytes apart); their product is hi hi + 2^-11 (hi lo + lo hi).  The two small parts are
// summed first, over the whole reduction, and scaled.
template <int SIZE, int ROWS, bool S, int WAVES>
struct GemmMover {
    static constexpr int SLAB = 128 / SIZE, CH = 16 / SIZE, COUNT = ROWS * 128 / 1024 / WAVES;
    static_assert(ROWS * 128 % (1024 * WAVES) == 0, "a wave moves whole kilobytes");
    uint32_t at[COUNT];                     // of the lane's chunks, from the slab's first byte on
    int along[COUNT];                       // their first reduction element in the slab
    const char *base; int64_t step;

    template <bool PAIRS>
    __device__ __forceinline__ void init(const void *p, int64_t ld, int64_t row0, int64_t rows, int lane, int wave)
    {
        const int left = (int)min((int64_t)ROWS, rows - row0);
        base = (const char *)p + (S ? row0 : row0 * ld) * SIZE;
        step = S ? SLAB * ld * SIZE : 128;
#pragma unroll
        for (int c = 0; c < COUNT; ++c) {
            const int pos = (c * WAVES + wave) * 64 + lane;                 // 16-byte place in the LDS tile
            if constexpr (S) {
                constexpr int PER = ROWS / 8;
                const int k = pos / PER, chunk = (gm_at_s<ROWS, PAIRS>(k, pos % PER) - k * (ROWS * 2)) >> 4;
                // columns past the operand's last are never stored: any of its values will do
                at[c] = (uint32_t)(k * ld * SIZE) + 16 * min(chunk, left / CH - 1);
                along[c] = k;
            } else {
                const int row = pos / 8, chunk = (gm_at_c<128, PAIRS>(row, pos % 8) - row * 128) >> 4;
                at[c] = (uint32_t)(min(row, left - 1) * ld * SIZE) + 16 * chunk;
                along[c] = chunk * CH;
            }
        }
    }
    // Transfer c of slab `index` of a plane that starts `plane` bytes after the first; `left` reduction elements exist from its first on.  What lies past them
    // is read as zeros: out of the buffer's range.  Written out (it has no output registers), because the compiler would have every transposing read wait
    // for all transfers before it, whatever their place; gm_arrive waits for the ones that matter, and orders reads against them.  Five wait states
    // between whatever wrote the descriptor (a spilled scalar comes back by a vector instruction) or m0, the place in LDS, and their use, which nobody else counts here.
    __device__ __forceinline__ void move(int c, int64_t index, int64_t plane, int64_t left, uint32_t tile, int wave) const
    {
        const uint64_t from = (uint64_t)(base + index * step + plane);
        const gm_i4 buffer = {(int)(uint32_t)from, (int)((uint32_t)(from >> 32) & 0xffffu), (int)0x80000000u, 0x00027000};
        const uint32_t v = along[c] < left ? at[c] : 0x80000000u;
        asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(v), "s"(buffer), "{m0}"(tile + (c * WAVES + wave) * 1024));
    }
};

// Waits until at most LEFT of the wave's transfers to LDS are on their way and its reads from LDS have ended, and for the other waves to get here.
template <int LEFT> __device__ __forceinline__ void gm_arrive() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory"); }

// Waves of 64 columns by 128 rows in tiles of 256 x 256, by 64 rows in smaller ones.
constexpr int gm_waves(int bm, int bn) { return bm * bn / 64 / (bm >= 256 ? 128 : 64); }
constexpr size_t gm_moved_lds(int bm, int bn) { return (size_t)2 * (bm + bn) * 128; }
// One tile of D.  lds: [2][BM + BN][128], which no wave reads any more.
template <int KIND, typename F, bool QS, bool PS, int BM, int BN, int PLANES>
__device__ __forceinline__ void gm_moved_tile(const GemmP &p, const F &f, int tm, int tn, int split, int64_t batch, char *lds)
{
    constexpr int WAVES = gm_waves(BM, BN), WP = BN / 64, TQ = BM / 16 / (WAVES / WP), SIZE = GemmKind<KIND>::size, SLAB = 128 / SIZE;
    constexpr int MOVES = (BM + BN) * 128 / 1024 / WAVES, HALF = (BM + BN) * 128;          // transfers of a wave, and bytes, a slab
    const int lane = fg_lane(), wave = fg_wave(), wp = wave % WP, tq0 = wave / WP * TQ;
    const int64_t once = (p.k + SLAB - 1) / SLAB, small = PLANES == 2 ? 2 * once : 0;       // slabs of the reduction, and of the small parts
    const int64_t per = p.slabs * (PLANES == 2 ? 3 : 1), s0 = split * per;
    const int slabs = (int)max((int64_t)0, min(once + small, s0 + per) - s0);
    constexpr bool PAIRS = F::W == 8;
    typename GemmKind<KIND>::acc acc[TQ][4] = {};
    GemmMover<SIZE, BM, QS, WAVES> q;
    GemmMover<SIZE, BN, PS, WAVES> b;
    q.template init<false>((const char *)p.q + batch * p.batch_q, p.ldq, (int64_t)tm * BM, p.rows_q, lane, wave);
    b.template init<PAIRS>((const char *)p.p + batch * p.batch_p, p.ldp, (int64_t)tn * BN, p.rows_p, lane, wave);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    // transfer c of slab i
    auto move = [&](int i, int c) {
        const int64_t s = s0 + i;
        const bool cross = PLANES == 2 && s < small;
        const int64_t at = cross ? s >> 1 : s - small, left = p.k - at * SLAB;
        const uint32_t to = lds0 + (i & 1) * HALF;
        if (c < q.COUNT) q.move(c, at, cross && (s & 1) ? p.plane_q : 0, left, to, wave);
        else b.move(c - q.COUNT, at, cross && !(s & 1) ? p.plane_p : 0, left, to + BM * 128, wave);
    };
    auto move_all = [&](int i) {
#pragma unroll
        for (int c = 0; c < MOVES; ++c) move(i, c);
    };
    struct Operands { gm_i4 a[4], b[TQ]; };
    // operand j of half h of slab i: four of P, then Q's
    auto read = [&](int i, int h, int j, Operands &o) {
        const char *from = lds + (i & 1) * HALF;
        if (j < 4) o.a[j] = gm_operand<128, BN, PS, PAIRS>(from + BM * 128, 4 * wp + j, h, lane);
        else o.b[j - 4] = gm_operand<128, BM, QS, false>(from, tq0 + j - 4, h, lane);
    };
    auto read_all = [&](int i, int h, Operands &o) {
#pragma unroll
        for (int j = 0; j < 4 + TQ; ++j) read(i, h, j, o);
    };
    auto multiply = [&](int t, int u, const Operands &o) { acc[t][u] = gm_mfma<KIND>(o.a[u], o.b[t], acc[t][u]); };
    auto scale = [&]() {
        if constexpr (PLANES == 2) {
#pragma unroll
            for (int t = 0; t < TQ; ++t)
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[t][u] *= 0x1p-11f;
        }
    };
    // Multiplies what `now` holds; reads half h of slab i into `next` and, where MOVE, starts the transfers of slab i + 1 on the way, spread over the instructions: a
    // compute unit takes a transfer every 16 cycles, and waves that begin with all of theirs wait for one another.
    auto half = [&]<bool MOVE>(int i, int h, const Operands &now, Operands &next) {
#pragma unroll
        for (int t = 0; t < TQ; ++t) {
            __builtin_amdgcn_sched_barrier(0);
            multiply(t, 0, now);
            multiply(t, 1, now);
            if constexpr (MOVE) {
#pragma unroll
                for (int c = t * MOVES / TQ; c < (t + 1) * MOVES / TQ; ++c) move(i + 1, c);
            }
#pragma unroll
            for (int j = t * (4 + TQ) / TQ; j < (t + 1) * (4 + TQ) / TQ; ++j) read(i, h, j, next);
            multiply(t, 2, now);
            multiply(t, 3, now);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    Operands first, second;
    if (slabs > 0) {
        move_all(0);
        if (slabs > 1) {
            move_all(1);
            gm_arrive<MOVES>();
        } else gm_arrive<0>();
        read_all(0, 0, first);
    }
    // nothing that came from scalar loads is on its way into the loop: they end in any order, and would turn every wait for LDS into one for all of it
    __builtin_amdgcn_s_waitcnt(0xc07f);
    int i = 0;
#pragma unroll 1
    for (; i + 2 < slabs; ++i) {
        if (PLANES == 2 && s0 + i == small) scale();
        half.template operator()<false>(i, 1, first, second);
        gm_arrive<0>();
        half.template operator()<true>(i + 1, 0, second, first);
    }
    // the last two, which start nothing any more
#pragma unroll 1
    for (; i < slabs; ++i) {
        if (PLANES == 2 && s0 + i == small) scale();
        half.template operator()<false>(i, 1, first, second);
        if (i + 1 < slabs) gm_arrive<0>();
        // (past the last slab: what is read is not used)
        half.template operator()<false>(i + 1, 0, second, first);
    }
    if (PLANES == 2 && s0 + slabs <= small) scale();
    gm_results<TQ>(p, f, batch, split, (int64_t)tm * BM + 16 * tq0, tn * BN + 64 * wp, lane, acc);
}
template <int KIND, typename F, bool QS, bool PS, int BM, int BN, int PLANES>
__global__ __launch_bounds__(64 * gm_waves(BM, BN), 2) void gemm_moved_kernel(GemmP p, F f)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int tm, tn, split;
    gm_tile(p, tm, tn, split);
    gm_moved_tile<KIND, F, QS, PS, BM, BN, PLANES>(p, f, tm, tn, split, blockIdx.y, lds);
}

// The same for two planes on a tile of 128 x 128, eight waves of 64 columns by 32 rows: a slab holds both planes of both operands and gives all three products (four
// parts moved for six), with sums of their own for the small ones.  Reductions that are short, or tiles that are few, wait for memory once a slab: a third
// as often.  lds: [2][4][128][128], which no wave reads any more.
constexpr size_t GM_PLANES_LDS = 2 * 4 * 128 * 128;
#define GM_PLANES_WAVES 8
template <typename F, bool QS, bool PS>
__device__ __forceinline__ void gm_planes_tile(const GemmP &p, const F &f, int tm, int tn, int split, int64_t batch, char *lds)
{
    constexpr int WAVES = GM_PLANES_WAVES, TQ = 2, PART = 128 * 128, HALF = 4 * PART;       // parts: Q hi, Q lo, P hi, P lo
    constexpr bool PAIRS = F::W == 8;
    const int lane = fg_lane(), wave = fg_wave(), wp = wave & 1, tq0 = (wave >> 1) * TQ;
    const int64_t s0 = split * p.slabs;
    const int slabs = (int)max((int64_t)0, min((p.k + 63) / 64, s0 + p.slabs) - s0);
    GemmMover<2, 128, QS, WAVES> q;
    GemmMover<2, 128, PS, WAVES> b;
    q.template init<false>((const char *)p.q + batch * p.batch_q, p.ldq, (int64_t)tm * 128, p.rows_q, lane, wave);
    b.template init<PAIRS>((const char *)p.p + batch * p.batch_p, p.ldp, (int64_t)tn * 128, p.rows_p, lane, wave);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    auto move = [&](int i) {
        const int64_t at = s0 + i, left = p.k - at * 64;
        const uint32_t to = lds0 + (i & 1) * HALF;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < q.COUNT; ++c) {
                q.move(c, at, h * p.plane_q, left, to + h * PART, wave);
                b.move(c, at, h * p.plane_p, left, to + (2 + h) * PART, wave);
            }
    };
    constexpr int MOVES = 4 * GemmMover<2, 128, QS, WAVES>::COUNT;
    gm_f4 acc[TQ][4] = {}, low[TQ][4] = {};
    if (slabs > 0) move(0);
    if (slabs > 1) move(1);
#pragma unroll 1
    for (int i = 0; i < slabs; ++i) {
        if (i + 1 < slabs) gm_arrive<MOVES>();
        else gm_arrive<0>();
        const char *from = lds + (i & 1) * HALF;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            gm_i4 a[2][4], x[2][TQ];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int u = 0; u < 4; ++u) a[e][u] = gm_operand<128, 128, PS, PAIRS>(from + (2 + e) * PART, 4 * wp + u, h, lane);
#pragma unroll
                for (int t = 0; t < TQ; ++t) x[e][t] = gm_operand<128, 128, QS, false>(from + e * PART, tq0 + t, h, lane);
            }
#pragma unroll
            for (int t = 0; t < TQ; ++t)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    acc[t][u] = gm_mfma<FGNN_F16>(a[0][u], x[0][t], acc[t][u]);
                    low[t][u] = gm_mfma<FGNN_F16>(a[1][u], x[0][t], low[t][u]);
                    low[t][u] = gm_mfma<FGNN_F16>(a[0][u], x[1][t], low[t][u]);
                }
        }
        if (i + 2 < slabs) {
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");     // this slab has been read everywhere
            move(i + 2);
        }
    }
#pragma unroll
    for (int t = 0; t < TQ; ++t)
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[t][u] += 0x1p-11f * low[t][u];
    gm_results<TQ>(p, f, batch, split, (int64_t)tm * 128 + 16 * tq0, tn * 128 + 64 * wp, lane, acc);
}
template <typename F, bool QS, bool PS>
__global__ __launch_bounds__(64 * GM_PLANES_WAVES, 2) void gemm_planes_kernel(GemmP p, F f)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int tm, tn, split;
    gm_tile(p, tm, tn, split);
    gm_planes_tile<F, QS, PS>(p, f, tm, tn, split, blockIdx.y, lds);
}

// ------------------------------------------------------------------------------------------------ few rows
// Products of at most 16 RT rows, bound by reading P once: a workgroup takes 16 CT columns of D, its waves share the reduction (blocks of four instructions' worth,
// 256 bytes of a row, dealt out in turn) and add up their sums in LDS.  Nothing is staged: a lane's 16 bytes of a row of P are its operand.
template <int KIND>
__device__ __forceinline__ void gm_rows_mfma(gm_i4 a, gm_i4 b, typename GemmKind<KIND>::acc &c)
{
    if constexpr (KIND == FGNN_F32) {
        const gm_f4 x = *(const gm_f4 *)&a, y = *(const gm_f4 *)&b;
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    } else if constexpr (KIND == FGNN_E4M3) {
        gm_i4 x[2], y[2];
        gm_widen(*(const uint32_t(*)[4])&a, x);
        gm_widen(*(const uint32_t(*)[4])&b, y);
#pragma unroll
        for (int j = 0; j < 2; ++j) c = gm_mfma<FGNN_F16>(x[j], y[j], c);
    } else c = gm_mfma<KIND>(a, b, c);
}
// 16 bytes at element k of a row of `left` + k elements, zeros past its end
template <int KIND>
__device__ __forceinline__ gm_i4 gm_rows_load(const char *p, int64_t left)
{
    constexpr int CH = 16 / GemmKind<KIND>::size;
    typedef int i4 __attribute__((ext_vector_type(4), aligned(1)));
    if (left >= CH) return *reinterpret_cast<const i4 *>(p);
    gm_i4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (i < left) {
            if constexpr (CH == 4) v[i] = ((const int *)p)[i];
            else if constexpr (CH == 8) v[i / 2] |= (int)((const uint16_t *)p)[i] << (16 * (i & 1));
            else v[i / 4] |= (int)((const uint8_t *)p)[i] << (8 * (i & 3));
        }
    return v;
}

#define GR_WAVES 8                          // most waves of a workgroup
template <int KIND, typename E, int RT, int CT>
__global__ __launch_bounds__(64 * GR_WAVES) void gemm_rows_kernel(GemmP p)
{
    constexpr int SIZE = GemmKind<KIND>::size, CH = 16 / SIZE, BLOCK = 256 / SIZE;
    typedef int i4 __attribute__((ext_vector_type(4), aligned(1)));
    typedef typename GemmKind<KIND>::acc acc_t;
    extern __shared__ __attribute__((aligned(16))) char lds[];                  // [waves][RT][CT][64] sums
    const int lane = fg_lane(), wave = fg_wave(), waves = (int)blockDim.x >> 6, r = lane & 15, g = lane >> 4, n0 = (int)blockIdx.x * 16 * CT;
    const char *w[CT], *x[RT];
#pragma unroll
    for (int c = 0; c < CT; ++c) w[c] = (const char *)p.p + (int64_t)min(n0 + 16 * c + r, p.n - 1) * p.ldp * SIZE + 16 * g;
#pragma unroll
    for (int t = 0; t < RT; ++t) x[t] = (const char *)p.q + min((int64_t)(16 * t + r), p.m - 1) * p.ldq * SIZE + 16 * g;
    acc_t acc[RT][CT] = {};
    const int64_t blocks = (p.k + BLOCK - 1) / BLOCK, whole = p.k / BLOCK;
    gm_i4 a[CT][4], b[RT][4];
    auto load = [&](int64_t blk) {
        const int64_t at = blk * 256;
        if (blk < whole) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int s = 0; s < 4; ++s) a[c][s] = *reinterpret_cast<const i4 *>(w[c] + at + 64 * s);
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int s = 0; s < 4; ++s) b[t][s] = *reinterpret_cast<const i4 *>(x[t] + at + 64 * s);
        } else {
            const int64_t left = p.k - blk * BLOCK - CH * g;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int c = 0; c < CT; ++c) a[c][s] = gm_rows_load<KIND>(w[c] + at + 64 * s, left - 4 * CH * s);
#pragma unroll
                for (int t = 0; t < RT; ++t) b[t][s] = gm_rows_load<KIND>(x[t] + at + 64 * s, left - 4 * CH * s);
            }
        }
    };
    int64_t blk = wave;
    if (blk < blocks) load(blk);
#pragma unroll 1
    for (; blk < blocks; blk += waves) {
        gm_i4 c[CT][4], d[RT][4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int i = 0; i < CT; ++i) c[i][s] = a[i][s];
#pragma unroll
            for (int t = 0; t < RT; ++t) d[t][s] = b[t][s];
        }
        if (blk + waves < blocks) load(blk + waves);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int i = 0; i < CT; ++i) gm_rows_mfma<KIND>(c[i][s], d[t][s], acc[t][i]);
    }
    acc_t *sums = (acc_t *)lds;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < CT; ++i) sums[((wave * RT + t) * CT + i) * 64 + lane] = acc[t][i];
    __syncthreads();
    for (int j = wave; j < RT * CT; j += waves) {
        acc_t s = sums[j * 64 + lane];
        for (int i = 1; i < waves; ++i) s += sums[(i * RT * CT + j) * 64 + lane];
        const int n = n0 + 16 * (j % CT) + 4 * g;
        GemmCols<4> cols;
        gm_columns(p.epi, min(n, p.n - 1), cols);
        float v[4] = {(float)s[0], (float)s[1], (float)s[2], (float)s[3]};
        gm_finish<E, 4>(p.epi, cols, gm_ahead<E, 4>(p.epi, 16 * (j / CT) + r, n), 16 * (j / CT) + r, n, v);
    }
}
