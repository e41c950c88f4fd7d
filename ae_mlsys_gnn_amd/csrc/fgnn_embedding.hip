// Rows of a table by tokens, y_i = s W[t_i], and the table's gradient dW[v] = s sum_{i: t_i = v} gy_i, summed in the tokens' order.
// Both are bound by memory.  The forward pass reads a row for every token.  For the gradient the tokens are sorted (stably, with their positions), and the sorted
// positions are cut into tiles of one length whatever the tokens, so that a token met a hundred thousand times is summed by as many workgroups as a hundred
// thousand tokens met once.  A token whose positions lie in one tile is written from there, beside workgroups that write zeros for the tokens that are not met; the parts of
// the others, two a tile at the most, are added up in a second launch.  Sums are 32 bits, in a fixed order.
#include <algorithm>
#include "fgnn_gemm.h"

#define EM_TPB 256
#define EM_GRID (1 << 20)
#define EM_FEW 4096                         // tokens that are sorted by their ranks
struct EmbeddingP {
    int64_t n; int vocabulary, cols;
    const void *tokens; int wide;           // wide: int64
    const void *w; int64_t ldw;
    float scale;
    void *y;
    const void *gy; int64_t ldg; void *dw;
    int lanes, groups, tiles_c;             // threads a row, rows a workgroup, parts of a row
    int length, tile; int64_t tiles;        // sorted positions of a group of threads and of a workgroup, workgroups' tiles
    const int *keys, *order;                // sorted tokens, their positions
    float *part;                            // [tiles][2][cols]: sums of the tile's first token (where it began before) and of its last (where it goes on)
};

__device__ __forceinline__ int64_t em_token(const EmbeddingP &p, int64_t i) { return p.wide ? ((const int64_t *)p.tokens)[i] : ((const int32_t *)p.tokens)[i]; }

template <typename E>
__global__ __launch_bounds__(EM_TPB) void embedding_kernel(EmbeddingP p)
{
    constexpr int V = fe_width<E>, U = 4;
    const int lane = (int)threadIdx.x % p.lanes, group = (int)threadIdx.x / p.lanes;
    const int64_t rows = (int64_t)p.groups * U, items = (p.n + rows - 1) / rows * p.tiles_c;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t i = item / p.tiles_c * rows + group;
        const int c = ((int)(item % p.tiles_c) * p.lanes + lane) * V;
        if (group >= p.groups || c >= p.cols) continue;
        float v[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = i + (int64_t)u * p.groups, t = at < p.n ? em_token(p, at) : 0;
            if (t >= 0 && t < p.vocabulary) gm_load<E, V>(v[u], (const E *)p.w + t * p.ldw + c, p.cols - c);
            else {
#pragma unroll
                for (int j = 0; j < V; ++j) v[u][j] = __builtin_nanf("");
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = i + (int64_t)u * p.groups;
            if (at >= p.n) break;
#pragma unroll
            for (int j = 0; j < V; ++j) v[u][j] *= p.scale;
            gm_store<E, V>(v[u], (E *)p.y + at * p.cols + c, p.cols - c);
        }
    }
}

// Tokens as 32-bit keys; those without a gradient (padding, outside the table) come last.
__device__ __forceinline__ int em_key(const EmbeddingP &p, int64_t i, int64_t padding)
{
    const int64_t t = em_token(p, i);
    return t >= 0 && t < p.vocabulary && t != padding ? (int)t : p.vocabulary;
}
__global__ __launch_bounds__(EM_TPB) void embedding_keys_kernel(EmbeddingP p, int64_t padding, int *__restrict__ keys)
{
    for (int64_t i = (int64_t)blockIdx.x * EM_TPB + threadIdx.x; i < p.n; i += (int64_t)gridDim.x * EM_TPB) keys[i] = em_key(p, i, padding);
}
// Few tokens are sorted by their ranks: EM_SHARE threads count what comes before a token, four comparisons a read of LDS (4096 tokens
// 15.5 us, 28 by digits in six launches; 8192 tokens 29, 29; with one thread a token 4096 took 140).
#define EM_SHARE 16
__global__ __launch_bounds__(EM_TPB) void embedding_rank_kernel(EmbeddingP p, int64_t padding, int *__restrict__ keys, int *__restrict__ order)
{
    __shared__ __attribute__((aligned(16))) int all[EM_FEW];
    const int n = (int)p.n, padded = (n + 3) & ~3;
    for (int i = threadIdx.x; i < padded; i += EM_TPB) all[i] = i < n ? em_key(p, i, padding) : 0x7fffffff;
    __syncthreads();
    const int i = (int)(blockIdx.x * (EM_TPB / EM_SHARE) + threadIdx.x / EM_SHARE), share = (int)threadIdx.x % EM_SHARE;
    const int key = all[min(i, n - 1)];
    int rank = 0;
#pragma unroll 4
    for (int j = 4 * share; j < padded; j += 4 * EM_SHARE) {
        const gm_i4 k = *reinterpret_cast<const gm_i4 *>(all + j);
#pragma unroll
        for (int u = 0; u < 4; ++u) rank += k[u] < key || (k[u] == key && j + u < i);
    }
#pragma unroll
    for (int o = EM_SHARE / 2; o > 0; o >>= 1) rank += __shfl_xor(rank, o, 64);
    if (i >= n || share) return;
    keys[rank] = key;
    order[rank] = i;
}
// The first sorted position of a key >= v, seven probes a step.
__device__ __forceinline__ int64_t em_bound(const int *__restrict__ keys, int64_t n, int v)
{
    int64_t lo = 0, hi = n;                 // keys[lo - 1] < v <= keys[hi]
    while (lo < hi) {
        const int64_t step = (hi - lo + 7) / 8;
        int below = 0;
#pragma unroll
        for (int j = 1; j < 8; ++j) {
            const int64_t at = lo + j * step - 1;
            below += at < hi && keys[at] < v;
        }
        // (keys are sorted: the first `below` probes are below v)
        hi = min(hi, below < 7 ? lo + (below + 1) * step - 1 : hi);
        lo += below * step;
    }
    return lo;
}

// A thread's channels in the gradient's sums: V of them, the last vector's moved back into the row (what it shares with the one before it is the same in both).
struct EmVector { int c, left; };           // left: 0 behind the last
template <int V>
__device__ __forceinline__ EmVector em_vector(const EmbeddingP &p, int tile, int lane)
{
    const int c = (tile * p.lanes + lane) * V;
    if (c >= p.cols) return {0, 0};
    const int from = p.cols >= V ? min(c, p.cols - V) : c;
    return {from, p.cols - from};
}
// V channels from c on of the U rows at(0), at(1) .. of gy, all of them asked for before one is converted (one after the other: 32,768 tokens of
// 50,257 rows of 1024 bf16 42 us, this way 32; 256 rows summed by one group 66, 33).
template <typename E, int V, int U, typename At>
__device__ __forceinline__ void em_rows(float (&v)[U][V], const EmbeddingP &p, int c, At at)
{
    typedef E vec __attribute__((ext_vector_type(V), aligned(sizeof(E))));
    const E *from[U];
#pragma unroll
    for (int u = 0; u < U; ++u) from[u] = (const E *)p.gy + (int64_t)at(u) * p.ldg + c;
    if (p.cols >= V) {
        vec raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = *reinterpret_cast<const vec *>(from[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) v[u][i] = (float)raw[u][i];
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) v[u][i] = i < p.cols ? (float)from[u][i < p.cols ? i : 0] : 0.f;
    }
}

// The first `tiles` x tiles_c workgroups sum tiles, the others write zeros for tokens that are not met, EM_ROWS of them each.
#define EM_ROWS 64
enum { EM_CLOSE = 1, EM_WHOLE = 2, EM_ON = 4 };
template <typename E>
__global__ __launch_bounds__(EM_TPB) void embedding_sum_kernel(EmbeddingP p)
{
    constexpr int V = fe_width<E>, U = 8;
    __shared__ float ends[2][EM_TPB * V];                       // a group's first token's sum, where it began before, and its last one's, where it goes on
    __shared__ int flags[EM_TPB], firsts[EM_TPB], lasts[EM_TPB];
    const int lane = (int)threadIdx.x % p.lanes, group = (int)threadIdx.x / p.lanes;
    if (blockIdx.x >= p.tiles * p.tiles_c) {
        const int row0 = (int)(blockIdx.x - p.tiles * p.tiles_c) * EM_ROWS, row = row0 + (int)threadIdx.x;
        if (threadIdx.x < EM_ROWS) {
            const int64_t at = row < p.vocabulary ? em_bound(p.keys, p.n, row) : 0;
            flags[threadIdx.x] = row < p.vocabulary && (at == p.n || p.keys[at] != row);
        }
        __syncthreads();
        const float zero[V] = {};
        for (int tile = 0; tile < p.tiles_c; ++tile)
            for (int r = group; r < EM_ROWS && group < p.groups; r += p.groups) {
                const int c = (tile * p.lanes + lane) * V;
                if (flags[r] && c < p.cols) gm_store<E, V>(zero, (E *)p.dw + (int64_t)(row0 + r) * p.cols + c, p.cols - c);
            }
        return;
    }
    const int64_t tile = blockIdx.x / p.tiles_c;
    const auto [c, left] = em_vector<V>(p, (int)(blockIdx.x % p.tiles_c), lane);
    const int64_t first = tile * p.tile + (int64_t)group * p.length, last = min(p.n, first + p.length);
    auto write = [&](float (&sum)[V], int key) {
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] *= p.scale;
        gm_store<E, V>(sum, (E *)p.dw + (int64_t)key * p.cols + c, left);
    };
    if (group < p.groups) {
        int flag = 0, now = first < last ? p.keys[first] : p.vocabulary;
        const int head = now;
        if (now < p.vocabulary) {
            bool open = first > 0 && p.keys[first - 1] == now;
            float sum[V];
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] = 0.f;
            auto keep = [&](int which) {
#pragma unroll
                for (int j = 0; j < V; ++j) ends[which][threadIdx.x * V + j] = sum[j];
            };
            for (int64_t i = first; i < last; i += U) {
                float g[U][V];
                int key[U];
#pragma unroll
                for (int u = 0; u < U; ++u) key[u] = p.keys[min(i + u, last - 1)];
                em_rows<E, V, U>(g, p, c, [&](int u) { return p.order[min(i + u, last - 1)]; });
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i + u >= last || now == p.vocabulary) break;
                    if (key[u] != now) {
                        if (open) {
                            keep(0);
                            flag |= EM_CLOSE;
                        } else if (left > 0) write(sum, now);
                        open = false;
                        now = key[u];
#pragma unroll
                        for (int j = 0; j < V; ++j) sum[j] = 0.f;
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) sum[j] += g[u][j];
                }
            }
            if (now < p.vocabulary) {
                const bool on = last < p.n && p.keys[last] == now;
                if (open || on) {
                    keep(open ? 0 : 1);
                    flag |= !open ? EM_ON : on ? EM_WHOLE : EM_CLOSE;
                } else if (left > 0) write(sum, now);
            }
        }
        if (lane == 0) {
            flags[group] = flag;
            firsts[group] = head;
            lasts[group] = now;
        }
    }
    __syncthreads();
    if (group != 0 || left <= 0) return;
    // the groups' ends in their order: a token that begins and ends in the workgroup's tile is written, the others' parts are kept
    float sum[V];
    int key = 0, have = 0;                  // have: 1 begun here, 2 before
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.f;
    for (int g = 0; g < p.groups; ++g) {
        const int flag = flags[g], from = (g * p.lanes + lane) * V;
        if (flag & (EM_CLOSE | EM_WHOLE)) {
            if (!have) {
                have = 2;
                key = firsts[g];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += ends[0][from + j];
            if (flag & EM_CLOSE) {
                if (have == 2) gm_store<float, V>(sum, p.part + 2 * tile * p.cols + c, left);
                else write(sum, key);
                have = 0;
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] = 0.f;
            }
        }
        if (flag & EM_ON) {
            have = 1;
            key = lasts[g];
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] = ends[1][from + j];
        }
    }
    if (have) gm_store<float, V>(sum, p.part + (2 * tile + (have == 1)) * p.cols + c, left);
}

// The same by a whole wave, 64 probes a step.
__device__ __forceinline__ int64_t em_bound_wave(const int *__restrict__ keys, int64_t n, int v)
{
    const int lane = fg_lane();
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t step = (hi - lo + 64) / 65, at = lo + (lane + 1) * step - 1;
        const int below = __popcll(__ballot(at < hi && keys[at < hi ? at : lo] < v));
        hi = min(hi, below < 64 ? lo + (below + 1) * step - 1 : hi);
        lo += below * step;
    }
    return lo;
}

// Tokens whose positions lie in more than one tile: the workgroup of the tile where they begin adds up their parts, its groups every so many of them, then those
// sums (one group for all of them: 124 parts of 128 fp32 took 40 us).
template <typename E>
__global__ __launch_bounds__(EM_TPB) void embedding_join_kernel(EmbeddingP p)
{
    constexpr int V = fe_width<E>;
    __shared__ float sums[EM_TPB * V];
    const int lane = (int)threadIdx.x % p.lanes, group = (int)threadIdx.x / p.lanes;
    const int64_t tile = blockIdx.x / p.tiles_c;
    const int c = ((int)(blockIdx.x % p.tiles_c) * p.lanes + lane) * V, left = p.cols - c;
    const int64_t first = tile * p.tile, end = first + p.tile;
    if (end >= p.n) return;
    const int key = p.keys[end - 1];
    if (key == p.vocabulary || p.keys[end] != key || (first > 0 && p.keys[first - 1] == key)) return;
    const int64_t last = (em_bound_wave(p.keys, p.n, key + 1) - 1) / p.tile;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.f;
    if (group < p.groups && left > 0) {
        if (group == 0) gm_load<float, V>(sum, p.part + (2 * tile + 1) * p.cols + c, left);
#pragma unroll 8
        for (int64_t t = tile + 1 + group; t <= last; t += p.groups) {
            float v[V];
            gm_load<float, V>(v, p.part + 2 * t * p.cols + c, left);
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += v[j];
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) sums[threadIdx.x * V + j] = sum[j];
    __syncthreads();
    if (group != 0 || left <= 0) return;
    for (int g = 1; g < p.groups; ++g)
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += sums[(g * p.lanes + lane) * V + j];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] *= p.scale;
    gm_store<E, V>(sum, (E *)p.dw + (int64_t)key * p.cols + c, left);
}

// As many tokens as a workgroup has threads, and a small table: everything in one launch without a workspace.  Every workgroup ranks them for itself and has `rows` tokens of the table, whose sums or
// zeros its groups write (239 tokens of 467 rows of 387 fp32, forward and backward: 45 us a call for 61.5, of which
// torch's hand-over of the backward pass takes 30).
template <typename E>
__global__ __launch_bounds__(EM_TPB) void embedding_few_kernel(EmbeddingP p, int64_t padding, int rows)
{
    constexpr int V = fe_width<E>;
    __shared__ __attribute__((aligned(16))) int all[EM_TPB];
    __shared__ int keys[EM_TPB], order[EM_TPB], starts[EM_ROWS + 1];
    const int n = (int)p.n, own = (int)threadIdx.x < n ? em_key(p, threadIdx.x, padding) : 0x7fffffff;
    all[threadIdx.x] = own;
    __syncthreads();
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 4) {
        const gm_i4 k = *reinterpret_cast<const gm_i4 *>(all + j);
#pragma unroll
        for (int u = 0; u < 4; ++u) rank += k[u] < own || (k[u] == own && j + u < (int)threadIdx.x);
    }
    if ((int)threadIdx.x < n) {
        keys[rank] = own;
        order[rank] = threadIdx.x;
    }
    __syncthreads();
    const int row0 = (int)(blockIdx.x / p.tiles_c) * rows;
    if ((int)threadIdx.x <= rows) starts[threadIdx.x] = (int)em_bound(keys, n, row0 + (int)threadIdx.x);
    __syncthreads();
    const int lane = (int)threadIdx.x % p.lanes, group = (int)threadIdx.x / p.lanes;
    const auto [c, left] = em_vector<V>(p, (int)(blockIdx.x % p.tiles_c), lane);
    if (group >= p.groups || left <= 0) return;
    for (int r = group; r < rows && row0 + r < p.vocabulary; r += p.groups) {
        float sum[V];
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.f;
        const int first = starts[r], last = starts[r + 1];
        auto add = [&]<int U>() {
            for (int i = first; i < last; i += U) {
                float g[U][V];
                em_rows<E, V, U>(g, p, c, [&](int u) { return order[min(i + u, last - 1)]; });
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < V; ++j) sum[j] += i + u < last ? g[u][j] : 0.f;
            }
        };
        if (last - first > 4) add.template operator()<16>();
        else add.template operator()<2>();
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] *= p.scale;
        gm_store<E, V>(sum, (E *)p.dw + (int64_t)(row0 + r) * p.cols + c, left);
    }
}

static void em_cut(EmbeddingP &p, int type)
{
    const int v = 16 / fe_size(type), vectors = (p.cols + v - 1) / v;
    p.tiles_c = (vectors + EM_TPB - 1) / EM_TPB;
    p.lanes = (vectors + p.tiles_c - 1) / p.tiles_c;
    p.groups = EM_TPB / p.lanes;
    p.length = 32;
    p.tile = p.length * p.groups;
    p.tiles = (p.n + p.tile - 1) / p.tile;
}

static bool em_limits(int64_t n, int vocabulary, int cols) { return n <= 2147483647LL - 65536 && vocabulary < 1 << 30 && cols <= 1 << 30; }
static int em_check(const char *who, int64_t n, int vocabulary, int cols, int type, const void *tokens, int wide)
{
    FGNN_REQUIRE(n >= 0 && vocabulary >= 0 && cols >= 1 && (wide == 0 || wide == 1) && fe_is_float(type), FGNN_ERR_SHAPE, "%s: bad sizes n=%lld vocabulary=%d cols=%d type=%d", who,
                 (long long)n, vocabulary, cols, type);
    FGNN_REQUIRE(em_limits(n, vocabulary, cols), FGNN_ERR_LIMIT, "%s: n=%lld vocabulary=%d cols=%d", who, (long long)n, vocabulary, cols);
    FGNN_REQUIRE(n == 0 || tokens, FGNN_ERR_NULL, "%s: NULL argument", who);
    return 0;
}

extern "C" int fgnn_embedding(int64_t n, int vocabulary, int cols, int type, const void *tokens, int wide, const void *weight, int64_t ldw, float scale, void *y, void *stream)
{
    const int rc = em_check("fgnn_embedding", n, vocabulary, cols, type, tokens, wide);
    if (rc || n == 0) return rc;
    FGNN_REQUIRE(ldw >= cols, FGNN_ERR_SHAPE, "fgnn_embedding: row stride %lld of %d columns", (long long)ldw, cols);
    FGNN_REQUIRE(y && (weight || vocabulary == 0), FGNN_ERR_NULL, "fgnn_embedding: NULL argument");
    EmbeddingP p = {n, vocabulary, cols, tokens, wide, weight, ldw, scale, y};
    em_cut(p, type);
    fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((embedding_kernel<E>), dim3((unsigned)std::min<int64_t>((n + 4 * p.groups - 1) / (4 * p.groups) * p.tiles_c, EM_GRID)), dim3(EM_TPB), 0, (hipStream_t)stream, p); });
    return fgnn_launch_status("embedding_kernel");
}

// Whether embedding_few_kernel does everything: few tokens, and a table of at most 16 MB, whose zeros take no longer than a call (100 MB: 54 us for 31).
static bool em_one(int64_t n, int vocabulary, int cols, int type) { return n > 0 && n <= EM_TPB && (int64_t)vocabulary * cols * fe_size(type) <= 1 << 24; }
// keys, order, the sums of the tiles' ends, the sort's own
struct EmbeddingSpace { size_t keys, part, sort; int bits; size_t all() const { return 3 * keys + part + sort; } };
static EmbeddingSpace em_space(const EmbeddingP &p)
{
    EmbeddingSpace s;
    s.bits = fgnn_rs_key_bits(p.vocabulary + 1);
    s.keys = fgnn_align256((size_t)p.n * sizeof(int));
    s.part = fgnn_align256((size_t)p.tiles * 2 * p.cols * sizeof(float));
    s.sort = p.n > EM_FEW ? fgnn_rs_sort_workspace(p.n, s.bits) : 0;
    return s;
}
extern "C" size_t fgnn_embedding_backward_workspace_bytes(int64_t n, int vocabulary, int cols, int type)
{
    if (n < 1 || vocabulary < 1 || cols < 1 || !em_limits(n, vocabulary, cols) || !fe_is_float(type) || em_one(n, vocabulary, cols, type)) return 0;
    EmbeddingP p = {n, vocabulary, cols};
    em_cut(p, type);
    return em_space(p).all();
}

extern "C" int fgnn_embedding_backward(int64_t n, int vocabulary, int cols, int type, const void *tokens, int wide, int64_t padding, const void *gy, int64_t ldg, float scale, void *dw,
                                       void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = em_check("fgnn_embedding_backward", n, vocabulary, cols, type, tokens, wide);
    if (rc || vocabulary == 0) return rc;
    FGNN_REQUIRE(ldg >= cols, FGNN_ERR_SHAPE, "fgnn_embedding_backward: row stride %lld of %d columns", (long long)ldg, cols);
    FGNN_REQUIRE(dw && (n == 0 || gy), FGNN_ERR_NULL, "fgnn_embedding_backward: NULL argument");
    EmbeddingP p = {n, vocabulary, cols, tokens, wide, nullptr, 0, scale, nullptr, gy, ldg, dw};
    em_cut(p, type);
    if (em_one(n, vocabulary, cols, type)) {
        // as many rows of the table a workgroup as leave four workgroups a compute unit: a row with tokens waits for memory, one without is only written
        const int cus = fgnn_current_device_compute_units(), rows = (int)std::min<int64_t>(EM_ROWS, std::max<int64_t>(p.groups, (int64_t)vocabulary * p.tiles_c / ((cus > 0 ? cus : 256) * 4)));
        const int64_t grid = ((int64_t)vocabulary + rows - 1) / rows * p.tiles_c;
        fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((embedding_few_kernel<E>), dim3((unsigned)grid), dim3(EM_TPB), 0, (hipStream_t)stream, p, padding, rows); });
        return fgnn_launch_status("embedding_few_kernel");
    }
    const EmbeddingSpace s = em_space(p);
    FGNN_REQUIRE(n == 0 || (workspace && workspace_bytes >= s.all()), FGNN_ERR_WORKSPACE, "fgnn_embedding_backward: workspace of %zu bytes", workspace_bytes);
    const int64_t summed = p.tiles * p.tiles_c, zeroed = ((int64_t)vocabulary + EM_ROWS - 1) / EM_ROWS;
    FGNN_REQUIRE(summed + zeroed < 1 << 24, FGNN_ERR_LIMIT, "fgnn_embedding_backward: n=%lld vocabulary=%d cols=%d", (long long)n, vocabulary, cols);
    hipStream_t st = (hipStream_t)stream;
    char *at = (char *)workspace;
    int *keys = (int *)at, *order = (int *)(at + s.keys);
    p.part = (float *)(at + 3 * s.keys);
    p.order = order;
    p.keys = keys;
    if (n > EM_FEW) {
        int *loose = (int *)(at + 2 * s.keys);
        hipLaunchKernelGGL(embedding_keys_kernel, dim3((unsigned)std::min<int64_t>((n + EM_TPB - 1) / EM_TPB, EM_GRID)), dim3(EM_TPB), 0, st, p, padding, loose);
        int launched = fgnn_launch_status("embedding_keys_kernel");
        if (launched) return launched;
        launched = fgnn_rs_sort_pairs(loose, nullptr, n, s.bits, order, &p.keys, at + 3 * s.keys + s.part, st);
        if (launched) return launched;
    } else if (n) hipLaunchKernelGGL(embedding_rank_kernel, dim3((unsigned)((n + EM_TPB / EM_SHARE - 1) / (EM_TPB / EM_SHARE))), dim3(EM_TPB), 0, st, p, padding, keys, order);
    fe_dispatch(type, [&]<typename E>() {
        hipLaunchKernelGGL((embedding_sum_kernel<E>), dim3((unsigned)(summed + zeroed)), dim3(EM_TPB), 0, st, p);
        if (p.tiles > 1) hipLaunchKernelGGL((embedding_join_kernel<E>), dim3((unsigned)summed), dim3(EM_TPB), 0, st, p);
    });
    return fgnn_launch_status("embedding_join_kernel");
}
