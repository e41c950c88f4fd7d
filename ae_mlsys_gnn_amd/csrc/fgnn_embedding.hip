// Rows of a table by tokens, y_i = s W[t_i], and the table's gradient dW[v] = s sum_{i: t_i = v} gy_i, summed in the tokens' order.
// Both are bound by memory.  The forward pass reads a row for every token.  For the gradient the tokens are sorted (stably, with their positions); the sorted
// positions are cut into tiles of one length whatever the tokens, so that a token met a hundred thousand times is summed by as many workgroups as a hundred
// thousand tokens met once.  A token whose positions lie in one tile is written from there; parts of the others are added up by the kernel that
// also writes the rows of tokens that are not met.  Sums are 32 bits, in a fixed order.
#include <algorithm>
#include "fgnn_gemm.h"

#define EM_TPB 256
#define EM_GRID (1 << 20)
struct EmbeddingP {
    int64_t n; int vocabulary, cols;
    const void *tokens; int wide;           // wide: int64
    const void *w; int64_t ldw;
    float scale;
    void *y;
    const void *gy; int64_t ldg; void *dw;
    int lanes, groups, tiles_c;             // threads a row, rows a workgroup, parts of a row
    int length; int64_t tiles;              // sorted positions a tile
    const int *keys, *order, *start;        // sorted tokens, their positions, where each token's begin [vocabulary + 1]
    float *part;                            // [tiles][2][cols]: sums of the tile's first token and of its last
};

__device__ __forceinline__ int64_t em_token(const EmbeddingP &p, int64_t i) { return p.wide ? ((const int64_t *)p.tokens)[i] : ((const int32_t *)p.tokens)[i]; }

template <typename E>
__global__ __launch_bounds__(EM_TPB) void embedding_kernel(EmbeddingP p)
{
    constexpr int V = fe_width<E>;
    const int lane = (int)threadIdx.x % p.lanes, group = (int)threadIdx.x / p.lanes;
    const int64_t items = (p.n + p.groups - 1) / p.groups * p.tiles_c;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t i = item / p.tiles_c * p.groups + group;
        const int c = ((int)(item % p.tiles_c) * p.lanes + lane) * V;
        if (group >= p.groups || i >= p.n || c >= p.cols) continue;
        const int64_t t = em_token(p, i);
        float v[V];
        if (t >= 0 && t < p.vocabulary) {
            gm_load<E, V>(v, (const E *)p.w + t * p.ldw + c, p.cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] *= p.scale;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = __builtin_nanf("");
        }
        gm_store<E, V>(v, (E *)p.y + i * p.cols + c, p.cols - c);
    }
}

// Tokens as 32-bit keys; those without a gradient (padding, outside the table) come last.
__global__ __launch_bounds__(EM_TPB) void embedding_keys_kernel(EmbeddingP p, int64_t padding, int *__restrict__ keys)
{
    for (int64_t i = (int64_t)blockIdx.x * EM_TPB + threadIdx.x; i < p.n; i += (int64_t)gridDim.x * EM_TPB) {
        const int64_t t = em_token(p, i);
        keys[i] = t >= 0 && t < p.vocabulary && t != padding ? (int)t : p.vocabulary;
    }
}
// start[v] = the first sorted position of a key >= v
__global__ __launch_bounds__(EM_TPB) void embedding_start_kernel(const int *__restrict__ keys, int64_t n, int vocabulary, int *__restrict__ start)
{
    const int v = (int)(blockIdx.x * EM_TPB + threadIdx.x);
    if (v > vocabulary) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < v) lo = mid + 1; else hi = mid;
    }
    start[v] = (int)lo;
}

template <typename E>
__global__ __launch_bounds__(EM_TPB) void embedding_sum_kernel(EmbeddingP p)
{
    constexpr int V = fe_width<E>, U = 8;
    const int lane = (int)threadIdx.x % p.lanes, group = (int)threadIdx.x / p.lanes;
    const int64_t items = (p.tiles + p.groups - 1) / p.groups * p.tiles_c;
    const int64_t end = p.start[p.vocabulary];                  // what lies behind has no gradient
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t tile = item / p.tiles_c * p.groups + group;
        const int c = ((int)(item % p.tiles_c) * p.lanes + lane) * V, left = p.cols - c;
        const int64_t first = tile * p.length, last = min(end, first + p.length);
        if (group >= p.groups || left <= 0 || first >= last) continue;
        float sum[V];
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.f;
        int now = p.keys[first];
        bool open = first > 0 && p.keys[first - 1] == now;      // the token's positions began in a tile before
        auto leave = [&](bool on) {                             // on: they go on behind this tile
            if (open || on) {
                gm_store<float, V>(sum, p.part + (2 * tile + (open ? 0 : 1)) * p.cols + c, left);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] *= p.scale;
                gm_store<E, V>(sum, (E *)p.dw + (int64_t)now * p.cols + c, left);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] = 0.f;
            open = false;
        };
        for (int64_t i = first; i < last; i += U) {
            float g[U][V];
            int key[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = min(i + u, last - 1);
                key[u] = p.keys[at];
                gm_load<E, V>(g[u], (const E *)p.gy + (int64_t)p.order[at] * p.ldg + c, left);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u >= last) break;
                if (key[u] != now) {
                    leave(false);
                    now = key[u];
                }
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += g[u][j];
            }
        }
        leave(last < end && p.keys[last] == now);
    }
}

// Rows of tokens that are not met, and of those whose positions lie in more than one tile: the first one's sum is its last token's, the others' their first's.
template <typename E>
__global__ __launch_bounds__(EM_TPB) void embedding_rows_kernel(EmbeddingP p)
{
    constexpr int V = fe_width<E>;
    const int lane = (int)threadIdx.x % p.lanes, group = (int)threadIdx.x / p.lanes;
    const int64_t items = ((int64_t)p.vocabulary + p.groups - 1) / p.groups * p.tiles_c;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t row = item / p.tiles_c * p.groups + group;
        const int c = ((int)(item % p.tiles_c) * p.lanes + lane) * V, left = p.cols - c;
        if (group >= p.groups || left <= 0 || row >= p.vocabulary) continue;
        const int64_t a = p.n ? p.start[row] : 0, b = p.n ? p.start[row + 1] : 0;
        float sum[V];
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] = 0.f;
        if (b > a) {
            const int64_t t0 = a / p.length, t1 = (b - 1) / p.length;
            if (t0 == t1) continue;
            // (it begins its first tile where a is the tile's first position: then that tile's sum is of its first token, and not open; see leave)
            gm_load<float, V>(sum, p.part + (2 * t0 + 1) * p.cols + c, left);
#pragma unroll 4
            for (int64_t t = t0 + 1; t <= t1; ++t) {
                float v[V];
                gm_load<float, V>(v, p.part + 2 * t * p.cols + c, left);
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] += v[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] *= p.scale;
        }
        gm_store<E, V>(sum, (E *)p.dw + row * p.cols + c, left);
    }
}

static void em_cut(EmbeddingP &p, int type)
{
    const int v = 16 / fe_size(type), vectors = (p.cols + v - 1) / v;
    p.tiles_c = (vectors + EM_TPB - 1) / EM_TPB;
    p.lanes = (vectors + p.tiles_c - 1) / p.tiles_c;
    p.groups = EM_TPB / p.lanes;
    p.length = 32;
    p.tiles = (p.n + p.length - 1) / p.length;
}
static unsigned em_grid(int64_t rows, const EmbeddingP &p) { return (unsigned)std::min<int64_t>((rows + p.groups - 1) / p.groups * p.tiles_c, EM_GRID); }

static int em_check(const char *who, int64_t n, int vocabulary, int cols, int type, const void *tokens, int wide)
{
    FGNN_REQUIRE(n >= 0 && vocabulary >= 0 && cols >= 1 && (wide == 0 || wide == 1) && fe_is_float(type), FGNN_ERR_SHAPE, "%s: bad sizes n=%lld vocabulary=%d cols=%d type=%d", who,
                 (long long)n, vocabulary, cols, type);
    FGNN_REQUIRE(n <= 2147483647LL - 65536 && vocabulary < 1 << 30 && cols <= 1 << 30, FGNN_ERR_LIMIT, "%s: n=%lld vocabulary=%d cols=%d", who, (long long)n, vocabulary, cols);
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
    fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((embedding_kernel<E>), dim3(em_grid(n, p)), dim3(EM_TPB), 0, (hipStream_t)stream, p); });
    return fgnn_launch_status("embedding_kernel");
}

// keys, order, start, the sums of the tiles' ends, the sort's own
struct EmbeddingSpace { size_t keys, start, part, sort; int bits; size_t all() const { return 2 * keys + start + part + sort; } };
static EmbeddingSpace em_space(const EmbeddingP &p)
{
    EmbeddingSpace s;
    s.bits = fgnn_rs_key_bits(p.vocabulary + 1);
    s.keys = fgnn_align256((size_t)p.n * sizeof(int));
    s.start = fgnn_align256(((size_t)p.vocabulary + 1) * sizeof(int));
    s.part = fgnn_align256((size_t)p.tiles * 2 * p.cols * sizeof(float));
    s.sort = fgnn_rs_sort_workspace(p.n, s.bits);
    return s;
}
extern "C" size_t fgnn_embedding_backward_workspace_bytes(int64_t n, int vocabulary, int cols, int type)
{
    if (n < 1 || vocabulary < 1 || vocabulary >= 1 << 30 || cols < 1 || !fe_is_float(type)) return 0;
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
    hipStream_t st = (hipStream_t)stream;
    if (n == 0) {
        fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((embedding_rows_kernel<E>), dim3(em_grid(vocabulary, p)), dim3(EM_TPB), 0, st, p); });
        return fgnn_launch_status("embedding_rows_kernel");
    }
    const EmbeddingSpace s = em_space(p);
    FGNN_REQUIRE(workspace && workspace_bytes >= s.all(), FGNN_ERR_WORKSPACE, "fgnn_embedding_backward: workspace of %zu bytes", workspace_bytes);
    char *at = (char *)workspace;
    int *keys = (int *)at, *order = (int *)(at + s.keys), *start = (int *)(at + 2 * s.keys);
    p.part = (float *)(at + 2 * s.keys + s.start);
    const unsigned flat = (unsigned)std::min<int64_t>((n + EM_TPB - 1) / EM_TPB, EM_GRID);
    hipLaunchKernelGGL(embedding_keys_kernel, dim3(flat), dim3(EM_TPB), 0, st, p, padding, keys);
    int launched = fgnn_launch_status("embedding_keys_kernel");
    if (launched) return launched;
    launched = fgnn_rs_sort_pairs(keys, nullptr, n, s.bits, order, &p.keys, at + 2 * s.keys + s.start + s.part, st);
    if (launched) return launched;
    p.order = order;
    p.start = start;
    hipLaunchKernelGGL(embedding_start_kernel, dim3((unsigned)(vocabulary / EM_TPB + 1)), dim3(EM_TPB), 0, st, p.keys, n, vocabulary, start);
    fe_dispatch(type, [&]<typename E>() {
        hipLaunchKernelGGL((embedding_sum_kernel<E>), dim3(em_grid(p.tiles, p)), dim3(EM_TPB), 0, st, p);
        hipLaunchKernelGGL((embedding_rows_kernel<E>), dim3(em_grid(vocabulary, p)), dim3(EM_TPB), 0, st, p);
    });
    return fgnn_launch_status("embedding_rows_kernel");
}
