// Attention of queries to keys and values of another length, softmax over the keys that are seen:
//   S = scale Q K^T,   P = exp(S - lse),   Y = P V,   lse = log sum exp S over the keys that are seen,
// and its gradient,  dV = P^T G,   dP = G V^T,   dS = P (dP - delta),   delta = rowsum(G Y),   dQ = scale dS K,   dK = scale dS^T Q.
// Nothing of the size of S is written: scores are formed tile by tile, and again in the backward pass.
//
// Every product is a matrix instruction of 32 x 32 sums whose second operand waits in registers. A wave owns 32 columns (queries in the forward pass and in that of dQ, keys
// in that of dK and dV) and walks tiles of the other side, which the workgroup's waves share in LDS.  Its scores come out with a lane per column and 16 of 32 rows in
// its registers (row 8 (i / 4) + 4 (lane / 32) + i % 4 in register i), so that a softmax is a matter of the lane and the one 32 lanes away, and the scores are,
// rounded, the second operand of the next product as they lie: the order of a reduction is free as long as both operands have the same, and the first operand, the tile
// transposed, is read from LDS in that order.
//
// 16-bit types: products of 16-bit values, P and dS rounded to the type (as the values they are multiplied with are), sums, statistics and results in 32 bits.  fp32: every
// operand in three planes of 8 significant bits (bf16, truncated, so that they add up to it exactly), and the six products that reach above 2^-24 of the result, small ones
// first: the matrix unit does 16 of them in the time of one fp32 product.  Infinities in fp32 operands have planes that are NaN.
#pragma once
#include "fgnn_gemm.h"

typedef float at_f16 __attribute__((ext_vector_type(16)));

struct AttentionP {
    int batch, nq, nk, heads, kv_heads, share, dim;             // share: heads that use the same keys
    int rows;                                                   // queries of one head of keys: nq share, row = position share + head
    uint32_t share_mul; int share_shift;                        // row / share
    const void *q, *k, *v, *g; int64_t qb, qn, qh, kb, kn, kh, vb, vn, vh, gb, gn, gh;      // strides of samples, positions and heads, in elements
    const void *lengths; int wide; const uint8_t *mask;         // keys seen: the first lengths[b], and those with mask[b][key]; NULL: all
    float scale, log2_scale;                                    // log2_scale = scale log2 e
    void *y; float *lse, *delta;                                // y [batch][nq][heads][dim]; [batch][heads][nq], lse in powers of two; +inf of rows that see nothing
    void *rest;                                                 // as y, of 16-bit types, NULL: not kept: what their rounding leaves, for delta
    void *dq, *dk, *dv;                                         // contiguous, as y
    int tiles, splits, per;                                     // tiles of 32 waves columns; parts of the other side, and tiles of each
    float *part, *part_lse;                                     // sums of the parts
};

// Planes of an operand, as 16-bit values; rows of a tile that lies in LDS.
template <typename E> constexpr int at_planes = sizeof(E) == 4 ? 3 : 1;
template <typename E> constexpr int at_tile = sizeof(E) == 4 ? 32 : 64;
constexpr int AT_CHUNK = 8;                 // components of 16 bytes of a plane

// 16-byte chunk `ch` of row `row` in a plane of ROW bytes a row.  LDS has 64 banks of four bytes: chunks are exchanged so that the reads meet each of them once, sixteen rows at
// one chunk, and four rows at four chunks next to one another.  What is exchanged is linear in the row's bits.
template <int ROW>
__host__ __device__ constexpr int at_exchange(int row)
{
    static_assert(ROW % 128 == 0, "whole lines of 32 banks a row");
    if (ROW % 256) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
    return (row & 3) << 2 | ((row >> 2) & 3);
}
template <int ROW>
__device__ __forceinline__ int at_place(int row, int ch) { return row * ROW + ((ch ^ at_exchange<ROW>(row)) << 4); }

// Where a lane reads planes of DP components: its row's first chunk for scores, and the first of what the reads of the transposed tile below say.  The others' places differ from
// these in bits of the chunk index that are exchanged (an exclusive or with a constant; eight registers for as many places and the sums of dK and dV left no room for two waves)
// and in constant offsets.
template <typename T> __device__ __forceinline__ auto at_lds(uint32_t at) { return (__attribute__((address_space(3))) T *)(uintptr_t)at; }
template <int DP>
struct AtReader {
    static constexpr int ROW = DP * 2, STEPS = ROW / 32, MASK = ROW % 256 ? 7 : 15;     // STEPS: instructions of a score; MASK: exchanged bits of the chunk index
    uint32_t score, gather;
    __device__ __forceinline__ void init(int lane)
    {
        const int h = lane >> 5, r = lane & 15;
        score = at_place<ROW>(lane & 31, h);
        // row 4 h + r / 4, four components from 16 ((lane / 16) % 2) + 4 (r % 4) on
        gather = at_place<ROW>(4 * h + (r >> 2), 2 * ((lane >> 4) & 1) + ((r & 3) >> 1)) + (r & 1) * 8;
    }
    // `from` (of a plane that starts at a multiple of 256 bytes), `chunks` chunks and `rows` rows further on; both constants, of bits that the lanes' own do not have
    static __device__ __forceinline__ uint32_t to(uint32_t from, int chunks, int rows) { return (from ^ (((chunks & MASK) ^ at_exchange<ROW>(rows)) << 4)) + (chunks & ~MASK) * 16 + rows * ROW; }
};

template <typename E>
__device__ __forceinline__ at_f16 at_multiply(gm_i4 a, gm_i4 b, at_f16 c)
{
    if constexpr (std::is_same_v<E, _Float16>) return __builtin_amdgcn_mfma_f32_32x32x16_f16(*(gm_h8 *)&a, *(gm_h8 *)&b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(gm_b8 *)&a, *(gm_b8 *)&b, c, 0, 0, 0);
}
// The products of two operands' planes
template <typename E, int P>
__device__ __forceinline__ at_f16 at_planes_multiply(const gm_i4 (&a)[P], const gm_i4 (&b)[P], at_f16 c)
{
#pragma unroll
    for (int s = P - 1; s >= 0; --s)
#pragma unroll
        for (int h = 0; h <= s; ++h) c = at_multiply<E>(a[s - h], b[h], c);
    return c;
}
// Columns as second operands: [STEPS][planes]
template <typename E, int DP> struct AtColumns { gm_i4 c[AtReader<DP>::STEPS][at_planes<E>]; };

// The scores of 32 rows of a tile (from row0 on, a multiple of 32) with the wave's columns.  plane: bytes from a plane to the next.
template <typename E, int DP>
__device__ __forceinline__ at_f16 at_scores(const AtReader<DP> &at, uint32_t tile, int plane, int row0, const AtColumns<E, DP> &cols)
{
    typedef AtReader<DP> R;
    constexpr int P = at_planes<E>;
    at_f16 s = {};
#pragma unroll
    for (int j = 0; j < R::STEPS; ++j) {
        gm_i4 a[P];
#pragma unroll
        for (int h = 0; h < P; ++h) a[h] = *at_lds<gm_i4>(R::to(tile + at.score, 2 * j, row0) + h * plane);
        s = at_planes_multiply<E, P>(a, cols.c[j], s);
    }
    return s;
}
// The same with the columns, of one plane, in LDS too, from `cols` on.
template <typename E, int DP>
__device__ __forceinline__ at_f16 at_scores(const AtReader<DP> &at, uint32_t tile, int row0, uint32_t cols)
{
    typedef AtReader<DP> R;
    at_f16 s = {};
#pragma unroll
    for (int j = 0; j < R::STEPS; ++j) s = at_multiply<E>(*at_lds<gm_i4>(R::to(tile + at.score, 2 * j, row0)), *at_lds<gm_i4>(R::to(cols + at.score, 2 * j, 0)), s);
    return s;
}

// 16 of a column's 32 weights as second operands: rounded to the type, or in planes.
template <typename E> struct AtWeights {
    gm_i4 w[2][at_planes<E>];
    __device__ __forceinline__ explicit AtWeights(const float (&v)[16])
    {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if constexpr (sizeof(E) == 4) {
                uint32_t bits[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) bits[i] = __float_as_uint(v[8 * s + i]);
                gm_split(bits, w[s]);
            } else {
                typedef E e8 __attribute__((ext_vector_type(8)));
                e8 b;
#pragma unroll
                for (int i = 0; i < 8; ++i) b[i] = (E)v[8 * s + i];
                w[s][0] = *(const gm_i4 *)&b;
            }
        }
    }
};
// acc[t] (32 components from 32 t on, by the wave's columns) += (32 rows of a tile, from row0 on)^T w
template <typename E, int DP>
__device__ __forceinline__ void at_gather(const AtReader<DP> &at, uint32_t tile, int plane, int row0, const AtWeights<E> &weights, at_f16 (&acc)[DP / 32])
{
    typedef AtReader<DP> R;
    constexpr int P = at_planes<E>;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) {
            // the transposing read: 16 lanes give four rows of 16 values (four a lane) and get a column of four each
            typedef short s8 __attribute__((ext_vector_type(8)));
            gm_i4 a[P];
#pragma unroll
            for (int h = 0; h < P; ++h) {
                const gm_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at_lds<gm_s4>(R::to(tile + at.gather, 4 * t, row0 + 16 * s) + h * plane));
                const gm_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at_lds<gm_s4>(R::to(tile + at.gather, 4 * t, row0 + 16 * s + 8) + h * plane));
                const s8 u = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                a[h] = *(const gm_i4 *)&u;
            }
            acc[t] = at_planes_multiply<E, P>(a, weights.w[s], acc[t]);
        }
}

// Asks that the matrix instructions of the code around it come for N operands from LDS one after the other, their reads (READS for each plane) AHEAD of them before the first (left
// alone the compiler reads each operand right before its instruction and waits for it), and in the shadow of each operand's VALU instructions of other arithmetic and EXPS
// exponentials.
template <int N, int PLANES, int READS, int AHEAD, int VALU = 0, int EXPS = 0>
__device__ __forceinline__ void at_ahead()
{
    constexpr int R = READS * PLANES, M = PLANES * (PLANES + 1) / 2;
    __builtin_amdgcn_sched_group_barrier(0x100, R * AHEAD, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
        if (i < N - AHEAD) __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
        if (VALU) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
        if (EXPS) __builtin_amdgcn_sched_group_barrier(0x400, EXPS, 0);
    }
}

// Two tiles (keys and values, or queries and their gradients) on their way to LDS, one pair ahead of the one that is worked on.  Rows that are not wanted (bit not
// set) and components past the last are zeros: out of the buffer's range.
template <typename E, int ROWS, int DP, int WAVES>
struct AtFeed {
    static constexpr int SIZE = (int)sizeof(E), ROW = DP * 2, CH = ROW / 16, THREADS = 64 * WAVES, PLANE = ROWS * ROW, TILE = at_planes<E> * PLANE, WORDS = SIZE * AT_CHUNK / 16;
    static constexpr bool MOVED = SIZE == 2;                    // straight to LDS, into two places in turn; else through registers, where it is taken apart
    static constexpr int COUNT = ROWS * CH / THREADS, STEP = THREADS / CH;          // chunks a thread, and rows between them
    static constexpr int BYTES = (MOVED ? 2 : 1) * 2 * TILE;
    static_assert(ROWS * CH % THREADS == 0 && THREADS % CH == 0, "threads share a tile evenly");
    uint32_t lds; int row, ch, left;        // lds: address there; left: components
    gm_i4 w[MOVED ? 1 : 2][MOVED ? 1 : COUNT][WORDS];

    __device__ __forceinline__ void init(char *lds_, int dim)
    {
        lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds_;
        row = (int)threadIdx.x / CH;
        ch = (int)threadIdx.x % CH;
        if constexpr (MOVED) ch ^= at_exchange<ROW>(row);       // the chunk that belongs where the thread's first transfer ends
        left = dim;
    }
    // The pair `index` from a and b on.
    __device__ __forceinline__ void start(int index, const void *a, const void *b, int64_t stride_a, int64_t stride_b, uint64_t bits)
    {
        constexpr uint64_t ALL = ROWS == 64 ? ~0ull : (1ull << ROWS) - 1;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const void *base = which ? b : a;
            const uint32_t step = (uint32_t)((which ? stride_b : stride_a) * SIZE);
            auto at = [&](int c, int word) {
                // (rows of a thread are a power of two apart: what is exchanged changes by a constant)
                const int chunk = MOVED ? ch ^ at_exchange<ROW>(c * STEP) : ch;
                const bool there = (bits == ALL || ((bits >> (row + c * STEP)) & 1)) && chunk * AT_CHUNK + word * (16 / SIZE) < left;
                return there ? (row + c * STEP) * step + (chunk * WORDS + word) * 16 : 0x80000000u;
            };
            if constexpr (MOVED) {
                // (written out, and its waits with it: see GemmMover)
                const uint64_t from = (uint64_t)base;
                const gm_i4 buffer = {(int)(uint32_t)from, (int)((uint32_t)(from >> 32) & 0xffffu), (int)0x80000000u, 0x00027000};
                const uint32_t to = lds + ((index & 1) * 2 + which) * TILE + fg_wave() * 1024;
#pragma unroll
                for (int c = 0; c < COUNT; ++c)
                    asm volatile("s_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(at(c, 0)), "s"(buffer), "{m0}"(to + c * THREADS * 16));
            } else {
                const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, 0x80000000u, 0x00027000);
#pragma unroll
                for (int c = 0; c < COUNT; ++c)
#pragma unroll
                    for (int i = 0; i < WORDS; ++i) w[which][c][i] = __builtin_amdgcn_raw_buffer_load_b128(from, at(c, i), 0, 0);
            }
        }
    }
    // The pair `index` has arrived, and nobody reads the one before any more.
    __device__ __forceinline__ uint32_t arrive(int index)
    {
        if constexpr (MOVED) {
            gm_arrive<0>();
            return lds + (index & 1) * 2 * TILE;
        } else {
            __syncthreads();
#pragma unroll
            for (int which = 0; which < 2; ++which)
#pragma unroll
                for (int c = 0; c < COUNT; ++c) {
                    uint32_t bits[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) bits[i] = (uint32_t)w[which][c][i / 4][i % 4];
                    gm_i4 part[3];
                    gm_split(bits, part);
#pragma unroll
                    for (int h = 0; h < 3; ++h) *at_lds<gm_i4>(lds + which * TILE + h * PLANE + at_place<ROW>(row + c * STEP, ch)) = part[h];
                }
            __syncthreads();
            return lds;
        }
    }
};

// A lane's components of one row, chunks 2 j + (lane / 32), zeros past the last and where the row is not there (`row` is memory that may be read all the same).  Any alignment;
// everything is asked for before anything is looked at (16 chunks one after the other: 2775 rows of 184 components in dQ's pass 56 us, this way 43).
template <typename E, int DP> struct AtWords { gm_i4 w[AtReader<DP>::STEPS][sizeof(E) * AT_CHUNK / 16]; };
template <typename E, int DP>
__device__ __forceinline__ void at_words(AtWords<E, DP> &words, const E *row, bool there, int dim, int lane)
{
    constexpr int V = fe_width<E>, N = AtReader<DP>::STEPS, WORDS = (int)sizeof(E) * AT_CHUNK / 16;
    if (dim % V == 0) {
        typedef typename fe_vec<E>::type vec;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                const int at = (2 * j + (lane >> 5)) * AT_CHUNK + w * V;
                const vec v = *reinterpret_cast<const vec *>(row + (at < dim ? at : 0));
                words.w[j][w] = *(const gm_i4 *)&v;
            }
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                const bool in = there && (2 * j + (lane >> 5)) * AT_CHUNK + w * V < dim;
#pragma unroll
                for (int i = 0; i < 4; ++i) words.w[j][w][i] = in ? words.w[j][w][i] : 0;
            }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const int at = (2 * j + (lane >> 5)) * AT_CHUNK + w * V + i;
                    const E v = row[at < dim ? at : 0];
                    ((E *)&words.w[j][w])[i] = there && at < dim ? v : (E)0.f;
                }
    }
}
// One row as the second operand of products.
template <typename E, int DP>
__device__ __forceinline__ void at_row(AtColumns<E, DP> &cols, const AtWords<E, DP> &words)
{
#pragma unroll
    for (int j = 0; j < AtReader<DP>::STEPS; ++j) {
        if constexpr (sizeof(E) == 4) {
            uint32_t bits[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) bits[i] = (uint32_t)words.w[j][i / 4][i % 4];
            gm_split(bits, cols.c[j]);
        } else cols.c[j][0] = words.w[j][0];
    }
}
template <typename E, int DP>
__device__ __forceinline__ void at_row(AtColumns<E, DP> &cols, const E *row, bool there, int dim, int lane)
{
    AtWords<E, DP> words;
    at_words<E, DP>(words, row, there, dim, lane);
    at_row<E, DP>(cols, words);
}
// Components of rows that the backward pass's operands hold: those that are not whole 16 bytes it has laid out anew, with zeros behind the last.
template <typename E> __device__ __forceinline__ int at_whole(int dim) { return (dim + fe_width<E> - 1) / fe_width<E> * fe_width<E>; }

// The value of the lane that holds the same column's other rows.
__device__ __forceinline__ float at_other_max(float v)
{
    const auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(u[0]), __uint_as_float(u[1]));
}
__device__ __forceinline__ float at_other_sum(float v)
{
    const auto u = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(u[0]) + __uint_as_float(u[1]);
}

// fp16 has 2^-14 as its smallest number of all significant bits, where softmax weights of long rows and gradients lie below: weights are rounded times 2^15
// (they are 1 at the most), gradients of scores times a power of two of the column's own that brings its largest so far to 2^14 .. 2^15.
template <typename E> constexpr float at_lift = std::is_same_v<E, _Float16> ? 15.f : 0.f;      // as an exponent
constexpr float AT_SLACK = 8.f;             // of the forward pass's maximum, as an exponent: its weights reach 2^8
template <typename E> constexpr float at_lift_forward = std::is_same_v<E, _Float16> ? 15.f - AT_SLACK : 0.f;
template <typename E, int STEPS>
struct AtRange {
    float f = std::is_same_v<E, _Float16> ? 0x1p96f : 1.f;
    __device__ __forceinline__ void fit(float (&w)[16], at_f16 (&acc)[STEPS])
    {
        if constexpr (std::is_same_v<E, _Float16>) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(w[i]));
            top = at_other_max(top);
            const bool over = top * f > 32768.f;
            if (__ballot(over)) {
                const float now = over ? __builtin_ldexpf(1.f, min(96, 15 - __builtin_amdgcn_frexp_expf(top))) : f, r = now / f;
                f = now;
#pragma unroll
                for (int t = 0; t < STEPS; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[t][i] *= r;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] *= f;
        }
    }
};

// What y's rounding to the type leaves, in the type (fp16, whose range ends at 2^-24, times 2^11, so that it lies below y and above that range as y does): delta is formed of both.
// Of the rounded y alone it is off by up to a half step of every component of Y, which does not cancel against dP where values share an offset (256 queries to 1024 keys of 64 bf16
// components, values of mean 4 and deviation 1: dQ was off by 1.8 % of its norm, this way by 0.25; a training step of 4 x 4096 queries takes 994 us, 976 without).
template <typename E> constexpr float at_rest_lift = std::is_same_v<E, _Float16> ? 2048.f : 1.f;
template <typename E>
__device__ __forceinline__ float at_rest(float y)
{
    const float rest = (y - (float)(E)y) * at_rest_lift<E>;
    return fabsf(rest) < __builtin_inff() ? rest : 0.f;        // (0 where y itself is no number of the type)
}
template <typename E> __device__ __forceinline__ float at_whole_y(E y, E rest) { return fmaf((float)rest, 1.f / at_rest_lift<E>, (float)y); }

// Which keys of a tile are seen.  The mask's bytes are asked for a tile ahead.
template <int TILE>
struct AtSeen {
    const uint8_t *mask; int64_t length; int lane;
    uint8_t next;
    __device__ __forceinline__ void init(const AttentionP &p, int b, int lane_)
    {
        lane = lane_;
        length = p.nk;
        if (p.lengths) {
            const int64_t n = p.wide ? ((const int64_t *)p.lengths)[b] : ((const int32_t *)p.lengths)[b];
            length = n < 0 ? 0 : n < p.nk ? n : p.nk;
        }
        mask = p.mask ? p.mask + (int64_t)b * p.nk : nullptr;
    }
    __device__ __forceinline__ void ask(int64_t key0) { if (mask) next = mask[min(key0 + lane, length - 1)]; }
    __device__ __forceinline__ uint64_t take(int64_t key0) const
    {
        const int64_t left = length - key0;
        if (mask) return __ballot(lane < TILE && lane < left && next);
        return left >= TILE ? (TILE == 64 ? ~0ull : (1ull << TILE) - 1) : left > 0 ? (1ull << left) - 1 : 0;
    }
};

// A workgroup's place.  Tiles of one head come one after the other and so on all XCDs at a time: where lengths differ, every XCD gets its share of the long ones (a head's
// tiles on one XCD, whose L2 then holds its keys: 4 x 4096 queries on 896 to 2048 keys, forward 322 us for 255).
struct AtPlace { int tile, split, head, b; };
__device__ __forceinline__ AtPlace at_block(const AttentionP &p)
{
    int t = (int)blockIdx.x;
    AtPlace o;
    o.tile = t % p.tiles;
    t /= p.tiles;
    o.split = t % p.splits;
    t /= p.splits;
    o.head = t % p.kv_heads;
    o.b = t / p.kv_heads;
    return o;
}
// Position and head of a row of queries.
__device__ __forceinline__ void at_query(const AttentionP &p, int row, int &pos, int &sub)
{
    pos = (int)((__umulhi((uint32_t)row, p.share_mul) + (uint32_t)row) >> p.share_shift);
    sub = row - pos * p.share;
}
// Where a row of queries lies in y or dq; NULL past the last.
template <typename E>
__device__ __forceinline__ E *at_result(const AttentionP &p, E *y, const AtPlace &o, int row)
{
    int pos, sub;
    at_query(p, row, pos, sub);
    return row < p.rows ? y + (((int64_t)o.b * p.nq + pos) * p.heads + o.head * p.share + sub) * p.dim : nullptr;
}
// A wave's sums, by `f`, to rows of `dim`: parts, in 32 bits, as they lie in the registers.
template <int DP, typename F>
__device__ __forceinline__ void at_store_part(const at_f16 (&acc)[DP / 32], float *row, int dim, int lane, F f)
{
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 32 * t + 8 * i + 4 * (lane >> 5);
            const float v[4] = {f(acc[t][4 * i]), f(acc[t][4 * i + 1]), f(acc[t][4 * i + 2]), f(acc[t][4 * i + 3])};
            if (d < dim) gm_store<float, 4>(v, row + d, dim - d);
        }
}
// Results, through the wave's own 32 rows of LDS from `lds` on, where a lane has four components of a row and leaves with 16 bytes next to its neighbours' (four
// components a lane are 16 bytes of each of 32 rows a store).  to(r): where row r of the wave's goes, NULL: nowhere.
template <typename E, int DP, typename F, typename To>
__device__ __forceinline__ void at_store(const at_f16 (&acc)[DP / 32], uint32_t lds, int dim, int lane, F f, To to)
{
    constexpr int V = fe_width<E>, SIZE = (int)sizeof(E), ROW = DP * SIZE, CH = ROW / 16;
    typedef E e4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 32 * t + 8 * i + 4 * (lane >> 5);
            const e4 v = {(E)f(acc[t][4 * i]), (E)f(acc[t][4 * i + 1]), (E)f(acc[t][4 * i + 2]), (E)f(acc[t][4 * i + 3])};
            *at_lds<e4>(lds + at_place<ROW>(lane & 31, d / V) + d % V * SIZE) = v;
        }
#pragma unroll
    for (int i = 0; i < CH / 2; ++i) {
        const int r = (i * 64 + lane) / CH, ch = (i * 64 + lane) % CH;
        typedef E vec __attribute__((ext_vector_type(V)));
        const vec u = *at_lds<vec>(lds + at_place<ROW>(r, ch));
        E *row = to(r), v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = u[j];
        if (row && ch * V < dim) gm_store<E, V>(v, row + ch * V, dim - ch * V);
    }
}
// LDS of a kernel: its feed's, or the results of all its waves.
template <typename E, int DP, int WAVES, int TILE> constexpr int at_bytes = std::max(AtFeed<E, TILE, DP, WAVES>::BYTES, WAVES * 32 * DP * (int)sizeof(E));

// Y and lse.  With `splits` parts of the keys, normalised sums and lse of each to `part`.
template <typename E, int DP, int WAVES, int TILE>
__global__ __launch_bounds__(64 * WAVES, DP > 128 ? 1 : 2) void attention_kernel(AttentionP p)
{
    constexpr int P = at_planes<E>, STEPS = AtReader<DP>::STEPS;
    extern __shared__ __attribute__((aligned(256))) char lds[];
    const AtPlace o = at_block(p);
    const int lane = fg_lane(), row = (o.tile * WAVES + fg_wave()) * 32 + (lane & 31);
    int pos, sub;
    at_query(p, min(row, p.rows - 1), pos, sub);
    const int head = o.head * p.share + sub;
    AtSeen<TILE> seen;
    seen.init(p, o.b, lane);
    const E *k = (const E *)p.k + o.b * p.kb + o.head * p.kh, *v = (const E *)p.v + o.b * p.vb + o.head * p.vh;
    AtColumns<E, DP> q;
    at_row<E, DP>(q, (const E *)p.q + o.b * p.qb + (int64_t)pos * p.qn + head * p.qh, row < p.rows, p.dim, lane);
    const int64_t first = (int64_t)o.split * p.per * TILE, last = min(seen.length, first + (int64_t)p.per * TILE);

    at_f16 acc[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) acc[t] = at_f16{};
    float most = -__builtin_inff(), sum = 0.f;
    typedef AtFeed<E, TILE, DP, WAVES> Feed;
    Feed feed;
    feed.init(lds, p.dim);
    AtReader<DP> at;
    at.init(lane);
    uint64_t bits = 0, coming = 0;
    if (first < last) {
        seen.ask(first);
        bits = seen.take(first);
        seen.ask(first + TILE);
        feed.start(0, k + first * p.kn, v + first * p.vn, p.kn, p.vn, bits);
    }
    int index = 0;
#pragma unroll 1
    for (int64_t key = first; key < last; key += TILE, bits = coming, ++index) {
        const uint32_t lk = feed.arrive(index), lv = lk + Feed::TILE;
        if (key + TILE < last) {
            coming = seen.take(key + TILE);
            seen.ask(key + 2 * TILE);
            feed.start(index + 1, k + (key + TILE) * p.kn, v + (key + TILE) * p.vn, p.kn, p.vn, coming);
        }
        if (bits == 0) continue;
        constexpr int B = TILE / 32;
        at_f16 s[B];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < B; ++t) s[t] = at_scores<E, DP>(at, lk, Feed::PLANE, 32 * t, q);
        at_ahead<B * STEPS, P, 1, P == 1 ? 4 : 2>();
        __builtin_amdgcn_sched_barrier(0);
        if (bits != (TILE == 64 ? ~0ull : (1ull << TILE) - 1)) {
#pragma unroll
            for (int t = 0; t < TILE / 32; ++t) {
                const uint32_t own = (uint32_t)(bits >> (32 * t)) >> (4 * (lane >> 5));
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = (own >> (8 * (i / 4) + i % 4)) & 1 ? s[t][i] : -__builtin_inff();
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < TILE / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
        top = at_other_max(top) * p.log2_scale;
        // Weights relative to a maximum that is too low by less than 2^8 are as exact and far from overflowing: only above that are sums and results scaled anew (one of 32
        // columns asks for a higher maximum in almost every tile of a short row), each column for itself, so that its result does not depend on its neighbours.
        const bool over = top > most + AT_SLACK;
        if (__ballot(over)) {
            const float now = over ? top : most, f = most > -__builtin_inff() ? __builtin_amdgcn_exp2f(most - now) : 0.f;
            most = now;
            sum *= f;
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][i] *= f;
        }
        const float base = (most > -__builtin_inff() ? most : 0.f) - at_lift_forward<E>;
        auto weigh = [&](int t) {
            float w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], p.log2_scale, -base));
                sum += w[i];
            }
            return AtWeights<E>(w);
        };
        AtWeights<E> w = weigh(0);
#pragma unroll
        for (int t = 0; t < B; ++t) {
            __builtin_amdgcn_sched_barrier(0);
            at_gather<E, DP>(at, lv, Feed::PLANE, 32 * t, w, acc);
            if (t + 1 < B) {
                w = weigh(t + 1);
                at_ahead<DP / 16, P, 2, P == 1 ? 3 : 1, 640 / DP, 256 / DP>();
            } else at_ahead<DP / 16, P, 2, P == 1 ? 3 : 1>();
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    sum = at_other_sum(sum);
    const bool none = sum == 0.f;
    const float inv = none ? 0.f : 1.f / sum;
    const auto norm = [&](float x) { return none ? 0.f : x * inv; };
    if (p.splits > 1) {
        if (row >= p.rows) return;
        const int64_t to = (((int64_t)o.b * p.kv_heads + o.head) * p.splits + o.split) * p.rows + row;
        at_store_part<DP>(acc, p.part + to * p.dim, p.dim, lane, norm);
        if (lane < 32) p.part_lse[to] = none ? -__builtin_inff() : most + __builtin_amdgcn_logf(sum) - at_lift_forward<E>;
        return;
    }
    if (p.lse && lane < 32 && row < p.rows) p.lse[((int64_t)o.b * p.heads + head) * p.nq + pos] = none ? __builtin_inff() : most + __builtin_amdgcn_logf(sum) - at_lift_forward<E>;
    __syncthreads();                        // the last tile has been read
    const uint32_t rows = feed.lds + fg_wave() * 32 * DP * (int)sizeof(E);
    at_store<E, DP>(acc, rows, p.dim, lane, norm, [&](int r) { return at_result(p, (E *)p.y, o, row - (lane & 31) + r); });
    if constexpr (sizeof(E) == 2) {
        if (p.rest) at_store<E, DP>(acc, rows, p.dim, lane, [&](float x) { return at_rest<E>(norm(x)); }, [&](int r) { return at_result(p, (E *)p.rest, o, row - (lane & 31) + r); });
    }
}

// dQ: as the forward pass, with P from lse.  With parts of the keys, their sums to `part`.  Forms delta = rowsum(G Y) of its rows, for itself and the pass of dK and dV.
template <typename E, int DP, int WAVES, int TILE>
__global__ __launch_bounds__(64 * WAVES, DP > (sizeof(E) == 4 ? 64 : 128) ? 1 : 2) void attention_dq_kernel(AttentionP p)
{
    constexpr int P = at_planes<E>, STEPS = AtReader<DP>::STEPS;
    extern __shared__ __attribute__((aligned(256))) char lds[];
    const AtPlace o = at_block(p);
    const int lane = fg_lane(), row = (o.tile * WAVES + fg_wave()) * 32 + (lane & 31);
    int pos, sub;
    at_query(p, min(row, p.rows - 1), pos, sub);
    const int head = o.head * p.share + sub;
    AtSeen<TILE> seen;
    seen.init(p, o.b, lane);
    const E *k = (const E *)p.k + o.b * p.kb + o.head * p.kh, *v = (const E *)p.v + o.b * p.vb + o.head * p.vh;
    AtColumns<E, DP> q, g;
    at_row<E, DP>(q, (const E *)p.q + o.b * p.qb + (int64_t)pos * p.qn + head * p.qh, row < p.rows, at_whole<E>(p.dim), lane);
    const int64_t stat = ((int64_t)o.b * p.heads + head) * p.nq + pos;
    const float lse = p.lse[stat] - at_lift<E>;
    float delta = 0.f;
    {
        AtWords<E, DP> y, rest = {}, up;
        const int64_t own = (((int64_t)o.b * p.nq + pos) * p.heads + head) * p.dim;
        at_words<E, DP>(up, (const E *)p.g + o.b * p.gb + (int64_t)pos * p.gn + head * p.gh, row < p.rows, at_whole<E>(p.dim), lane);
        at_words<E, DP>(y, (const E *)p.y + own, row < p.rows, p.dim, lane);
        if constexpr (sizeof(E) == 2) {
            if (p.rest) at_words<E, DP>(rest, (const E *)p.rest + own, row < p.rows, p.dim, lane);
        }
        at_row<E, DP>(g, up);
#pragma unroll
        for (int j = 0; j < STEPS; ++j)
#pragma unroll
            for (int i = 0; i < AT_CHUNK; ++i) delta = fmaf(at_whole_y(((const E *)y.w[j])[i], ((const E *)rest.w[j])[i]), (float)((const E *)up.w[j])[i], delta);
        delta = at_other_sum(delta);
        if (o.split == 0 && lane < 32 && row < p.rows) p.delta[stat] = delta;
    }
    AtRange<E, DP / 32> range;
    const int64_t first = (int64_t)o.split * p.per * TILE, last = min(seen.length, first + (int64_t)p.per * TILE);

    at_f16 acc[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) acc[t] = at_f16{};
    typedef AtFeed<E, TILE, DP, WAVES> Feed;
    Feed feed;
    feed.init(lds, p.dim);
    AtReader<DP> at;
    at.init(lane);
    uint64_t bits = 0, coming = 0;
    if (first < last) {
        seen.ask(first);
        bits = seen.take(first);
        seen.ask(first + TILE);
        feed.start(0, k + first * p.kn, v + first * p.vn, p.kn, p.vn, bits);
    }
    int index = 0;
#pragma unroll 1
    for (int64_t key = first; key < last; key += TILE, bits = coming, ++index) {
        const uint32_t lk = feed.arrive(index), lv = lk + Feed::TILE;
        if (key + TILE < last) {
            coming = seen.take(key + TILE);
            seen.ask(key + 2 * TILE);
            feed.start(index + 1, k + (key + TILE) * p.kn, v + (key + TILE) * p.vn, p.kn, p.vn, coming);
        }
        if (bits == 0) continue;
        constexpr int B = TILE / 32;
        at_f16 s[B], dp[B];
        float w[B][16];
        auto scores = [&](int t) {
            s[t] = at_scores<E, DP>(at, lk, Feed::PLANE, 32 * t, q);
            dp[t] = at_scores<E, DP>(at, lv, Feed::PLANE, 32 * t, g);
        };
        auto weigh = [&](int t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], p.log2_scale, -lse)) * (dp[t][i] - delta);
        };
        auto gather = [&](int t) {
            const uint32_t part = (uint32_t)(bits >> (32 * t));
            if (part != ~0u) {
                const uint32_t own = part >> (4 * (lane >> 5));
#pragma unroll
                for (int i = 0; i < 16; ++i) w[t][i] = (own >> (8 * (i / 4) + i % 4)) & 1 ? w[t][i] : 0.f;
            }
            range.fit(w[t], acc);
            at_gather<E, DP>(at, lk, Feed::PLANE, 32 * t, AtWeights<E>(w[t]), acc);
        };
        __builtin_amdgcn_sched_barrier(0);
        scores(0);
        at_ahead<2 * STEPS, P, 1, P == 1 ? 3 : 1>();
#pragma unroll
        for (int t = 0; t < B; ++t) {
            __builtin_amdgcn_sched_barrier(0);
            weigh(t);
            if (t + 1 < B) {                // the next keys' scores beside these ones' weights
                scores(t + 1);
                at_ahead<2 * STEPS, P, 1, P == 1 ? 3 : 1, 384 / DP, 128 / DP>();
            }
            __builtin_amdgcn_sched_barrier(0);
            gather(t);
            at_ahead<DP / 16, P, 2, P == 1 ? 3 : 1>();
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    const float f = p.scale / range.f * __builtin_amdgcn_exp2f(-at_lift<E>);
    const auto scaled = [&](float x) { return x * f; };
    if (p.splits > 1) {
        if (row >= p.rows) return;
        const int64_t to = (((int64_t)o.b * p.kv_heads + o.head) * p.splits + o.split) * p.rows + row;
        at_store_part<DP>(acc, p.part + to * p.dim, p.dim, lane, scaled);
        return;
    }
    __syncthreads();
    at_store<E, DP>(acc, feed.lds + fg_wave() * 32 * DP * (int)sizeof(E), p.dim, lane, scaled, [&](int r) { return at_result(p, (E *)p.dq, o, row - (lane & 31) + r); });
}

// dK and dV: a wave owns 32 keys and walks the queries of every head that uses them, tile by tile.  Where their sums leave no room in the registers the keys wait in LDS (their
// values stay): two waves a SIMD at 128 components, where one alone waits for LDS before every instruction.
constexpr bool at_keys_in_lds(int dim, int size) { return size == 2 && dim >= 128; }
// 32 rows a tile: three waves a SIMD at 64 components of 16 bits, where with 64 rows it is two (64 queries to 232,965 keys, 8 heads: 302 us for 262).
constexpr int AT_ROWS_DKV = 32;
template <typename E, int DP, int WAVES, int TILE>
__global__ __launch_bounds__(64 * WAVES, sizeof(E) == 4 ? 1 : DP > 128 ? 1 : DP > 64 ? 2 : 3) void attention_dkv_kernel(AttentionP p)
{
    constexpr int SIZE = (int)sizeof(E), P = at_planes<E>, STEPS = AtReader<DP>::STEPS, PARTS = DP / 32;
    constexpr bool KEYS_IN_LDS = at_keys_in_lds(DP, SIZE);
    extern __shared__ __attribute__((aligned(256))) char lds[];
    typedef AtFeed<E, TILE, DP, WAVES> Feed;
    const uint32_t stats = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + at_bytes<E, DP, WAVES, TILE>;       // lse, delta of the tile's rows, two tiles in turn
    const AtPlace o = at_block(p);
    const int lane = fg_lane(), key = (o.tile * WAVES + fg_wave()) * 32 + (lane & 31);
    AtSeen<64> seen;
    seen.init(p, o.b, lane);
    const bool there = key < seen.length && (!p.mask || seen.mask[min(key, p.nk - 1)]), any = __ballot(there) != 0;
    // tiles of every head's positions, one head after the other
    const int per_head = (p.nq + TILE - 1) / TILE, first = o.split * p.per;
    // (behind the last key that is seen nothing is walked)
    const int last = o.tile * WAVES * 32 < seen.length ? min(per_head * p.share, first + p.per) : first;

    at_f16 dk[PARTS], dv[PARTS];
#pragma unroll
    for (int t = 0; t < PARTS; ++t) dk[t] = dv[t] = at_f16{};
    AtRange<E, PARTS> range;
    Feed feed;
    feed.init(lds, p.dim);
    const uint32_t own_keys = stats + 4 * TILE * 4 + fg_wave() * 32 * AtReader<DP>::ROW;
    AtColumns<E, DP> k, v;
    if (first < last) {                     // (without a query nothing has been laid out anew)
        const int64_t own = min(key, p.nk - 1);
        at_row<E, DP>(k, (const E *)p.k + o.b * p.kb + own * p.kn + o.head * p.kh, there, at_whole<E>(p.dim), lane);
        at_row<E, DP>(v, (const E *)p.v + o.b * p.vb + own * p.vn + o.head * p.vh, there, at_whole<E>(p.dim), lane);
        if constexpr (KEYS_IN_LDS) {        // (read by their own wave alone)
#pragma unroll
            for (int j = 0; j < STEPS; ++j) *at_lds<gm_i4>(own_keys + at_place<AtReader<DP>::ROW>(lane & 31, 2 * j + (lane >> 5))) = k.c[j][0];
        }
    }
    AtReader<DP> at;
    at.init(lane);
    float stat = 0.f;
    auto fetch = [&](int i) {
        const int sub = i / per_head, pos = (i - sub * per_head) * TILE, head = o.head * p.share + sub, left = p.nq - pos;
        const uint64_t bits = left >= TILE ? (TILE == 64 ? ~0ull : (1ull << TILE) - 1) : (1ull << left) - 1;
        // rows past the last weigh nothing
        const int r = (int)threadIdx.x % TILE, which = (int)threadIdx.x / TILE;
        if (which < 2) stat = r < left ? (which ? p.delta : p.lse)[((int64_t)o.b * p.heads + head) * p.nq + pos + r] - (which ? 0.f : at_lift<E>) : which ? 0.f : __builtin_inff();
        feed.start(i - first, (const E *)p.q + o.b * p.qb + (int64_t)pos * p.qn + head * p.qh, (const E *)p.g + o.b * p.gb + (int64_t)pos * p.gn + head * p.gh, p.qn, p.gn, bits);
    };
    static_assert(64 * WAVES >= 2 * TILE, "a thread for every row's lse and delta");
    if (first < last) fetch(first);
#pragma unroll 1
    for (int i = first; i < last; ++i) {
        const uint32_t row_stats = stats + ((i - first) & 1) * 2 * TILE * 4;
        if (threadIdx.x < 2 * TILE) *at_lds<float>(row_stats + threadIdx.x * 4) = stat;
        const uint32_t lq = feed.arrive(i - first), lg = lq + Feed::TILE;
        if (i + 1 < last) fetch(i + 1);
        if (!any) continue;
#pragma unroll
        for (int t = 0; t < TILE / 32; ++t) {
            __builtin_amdgcn_sched_barrier(0);      // 32 rows at a time: the registers are full of sums
            at_f16 s;
            if constexpr (KEYS_IN_LDS) s = at_scores<E, DP>(at, lq, 32 * t, own_keys);
            else s = at_scores<E, DP>(at, lq, Feed::PLANE, 32 * t, k);
            const at_f16 dp = at_scores<E, DP>(at, lg, Feed::PLANE, 32 * t, v);
            at_ahead<2 * STEPS, P, 1, P == 1 ? 3 : 1>();
            __builtin_amdgcn_sched_barrier(0);
            float w[16], ds[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const gm_f4 lse = *at_lds<gm_f4>(row_stats + (32 * t + 8 * j + 4 * (lane >> 5)) * 4), delta = *at_lds<gm_f4>(row_stats + (TILE + 32 * t + 8 * j + 4 * (lane >> 5)) * 4);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    w[4 * j + c] = __builtin_amdgcn_exp2f(fmaf(s[4 * j + c], p.log2_scale, -lse[c]));
                    ds[4 * j + c] = w[4 * j + c] * (dp[4 * j + c] - delta[c]);
                }
            }
            range.fit(ds, dk);
            const AtWeights<E> pw(w), pd(ds);
            __builtin_amdgcn_sched_barrier(0);
            at_gather<E, DP>(at, lg, Feed::PLANE, 32 * t, pw, dv);
            at_gather<E, DP>(at, lq, Feed::PLANE, 32 * t, pd, dk);
            at_ahead<DP / 8, P, 2, P == 1 ? 3 : 1>();
        }
    }
    // keys that are not seen were zeros in every product: what a score of 0 made of them is dropped
    const float down = __builtin_amdgcn_exp2f(-at_lift<E>), f = p.scale / range.f * down;
    const auto sk = [&](float x) { return there ? x * f : 0.f; };
    const auto sv = [&](float x) { return there ? x * down : 0.f; };
    if (p.splits > 1) {
        if (key >= p.nk) return;
        const int64_t n = (int64_t)p.batch * p.nk * p.kv_heads * p.dim, to = o.split * 2 * n + (((int64_t)o.b * p.nk + key) * p.kv_heads + o.head) * p.dim;
        at_store_part<DP>(dk, p.part + to, p.dim, lane, sk);
        at_store_part<DP>(dv, p.part + to + n, p.dim, lane, sv);
        return;
    }
    __syncthreads();
    const auto to = [&](void *result, int r) {
        const int k = key - (lane & 31) + r;
        return k < p.nk ? (E *)result + (((int64_t)o.b * p.nk + k) * p.kv_heads + o.head) * p.dim : nullptr;
    };
    const uint32_t rows = feed.lds + fg_wave() * 32 * DP * SIZE;
    at_store<E, DP>(dk, rows, p.dim, lane, sk, [&](int r) { return to(p.dk, r); });
    at_store<E, DP>(dv, rows, p.dim, lane, sv, [&](int r) { return to(p.dv, r); });
}

// The kernels of a type, by what they are for: one file each (fgnn_attention_*.hip).
enum { AT_FORWARD, AT_DQ, AT_DKV };
struct AtShape { int waves, tile, dim; };                       // waves a workgroup, rows of a tile in LDS, padded components
template <typename E> void at_launch(int what, const AtShape &shape, const AttentionP &p, unsigned grid, hipStream_t st);

template <typename E, int DP>
static void at_launch_dim(int what, const AtShape &s, const AttentionP &p, unsigned grid, hipStream_t st)
{
    if (what == AT_DKV) {
        constexpr int S = (int)sizeof(E), R = AT_ROWS_DKV, bytes = at_bytes<E, DP, 4, R> + 4 * R * (int)sizeof(float) + (at_keys_in_lds(DP, S) ? 128 * DP * S : 0);
        hipLaunchKernelGGL((attention_dkv_kernel<E, DP, 4, R>), dim3(grid), dim3(256), bytes, st, p);
        return;
    }
    const auto queries = [&]<int WAVES, int TILE>() {
        constexpr int bytes = at_bytes<E, DP, WAVES, TILE>;
        if (what == AT_DQ) hipLaunchKernelGGL((attention_dq_kernel<E, DP, WAVES, TILE>), dim3(grid), dim3(64 * WAVES), bytes, st, p);
        else hipLaunchKernelGGL((attention_kernel<E, DP, WAVES, TILE>), dim3(grid), dim3(64 * WAVES), bytes, st, p);
    };
    if (s.waves == 4) queries.template operator()<4, at_tile<E>>();
    else if constexpr (sizeof(E) == 2 || DP <= 64) {
        if (s.waves == 2) queries.template operator()<2, 32>();
        else queries.template operator()<1, 32>();
    }
}
template <typename E>
void at_launch(int what, const AtShape &s, const AttentionP &p, unsigned grid, hipStream_t st)
{
    if (s.dim == 64) at_launch_dim<E, 64>(what, s, p, grid, st);
    else if (s.dim == 128) at_launch_dim<E, 128>(what, s, p, grid, st);
    else at_launch_dim<E, 256>(what, s, p, grid, st);
}
