// Attention: the C entries, the choice of tiles and parts, and the small kernels around those of fgnn_attention.h.
#include <algorithm>
#include "fgnn_attention.h"

#define AT_TPB 256
extern template void at_launch<float>(int, const AtShape &, const AttentionP &, unsigned, hipStream_t);
extern template void at_launch<__bf16>(int, const AtShape &, const AttentionP &, unsigned, hipStream_t);
extern template void at_launch<_Float16>(int, const AtShape &, const AttentionP &, unsigned, hipStream_t);

// delta = rowsum(G Y) where dQ, whose pass forms it by the way, is not wanted: two threads a row, summed as there.
template <typename E>
__global__ __launch_bounds__(AT_TPB) void attention_delta_kernel(AttentionP p)
{
    const int half = (int)threadIdx.x & 1;
    const int64_t rows = (int64_t)p.batch * p.nq * p.heads;
    for (int64_t first = (int64_t)blockIdx.x * (AT_TPB / 2); first < rows; first += (int64_t)gridDim.x * (AT_TPB / 2)) {
        const int64_t row = first + threadIdx.x / 2, pos = row / p.heads % p.nq, b = row / p.heads / p.nq;
        const int head = (int)(row % p.heads);
        float sum = 0.f;
        if (row < rows)
            for (int d = half * AT_CHUNK; d < p.dim; d += 2 * AT_CHUNK) {
                E y[AT_CHUNK], rest[AT_CHUNK] = {};
                float g[AT_CHUNK];
                gm_load<E, AT_CHUNK>(y, (const E *)p.y + row * p.dim + d, p.dim - d);
                if (p.rest) gm_load<E, AT_CHUNK>(rest, (const E *)p.rest + row * p.dim + d, p.dim - d);
                gm_load<E, AT_CHUNK>(g, (const E *)p.g + b * p.gb + pos * p.gn + head * p.gh + d, p.dim - d);
#pragma unroll
                for (int i = 0; i < AT_CHUNK; ++i) sum = fmaf(at_whole_y(y[i], rest[i]), g[i], sum);
            }
        sum += __shfl_xor(sum, 1, 64);
        if (row < rows && half == 0) p.delta[(b * p.heads + head) * p.nq + pos] = sum;
    }
}

// A workgroup's threads on rows of quads of components: `quads` threads (a power of two) a row and share of the parts, `shares` shares of a row's parts (a power of two),
// the rest rows side by side.
struct AtJoin { int quads, shares; int64_t rows; };
struct AtJoinPlace { int64_t row; int d, share; };
__device__ __forceinline__ AtJoinPlace at_join_place(const AtJoin &j)
{
    const int at = (int)threadIdx.x / j.quads;
    return {(int64_t)blockIdx.x * (AT_TPB / (j.quads * j.shares)) + at / j.shares, (int)threadIdx.x % j.quads * 4, at % j.shares};
}
// The shares' sums, in their order; true for the threads that have them all.
template <int N>
__device__ __forceinline__ bool at_join(const AtJoin &j, float (*sums)[AT_TPB], float (&v)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) sums[i][threadIdx.x] = v[i];
    __syncthreads();
    if (at_join_place(j).share) return false;
    for (int s = 1; s < j.shares; ++s)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += sums[i][threadIdx.x + s * j.quads];
    return true;
}

// Parts of the keys joined: Y = sum 2^(lse_s - lse) Y_s over the parts, in a fixed order.
template <typename E>
__global__ __launch_bounds__(AT_TPB) void attention_join_kernel(AttentionP p, AtJoin j)
{
    __shared__ float sums[5][AT_TPB];
    const AtJoinPlace o = at_join_place(j);
    const int64_t group = o.row / p.rows, b = group / p.kv_heads;
    const int row = (int)(o.row - group * p.rows), pos = row / p.share, head = (int)(group % p.kv_heads) * p.share + row % p.share;
    const bool there = o.row < j.rows;
    const int64_t at = group * p.splits * p.rows + row;
    float most = -__builtin_inff(), v[5] = {};
    if (there)
        for (int s = o.share; s < p.splits; s += j.shares) most = fmaxf(most, p.part_lse[at + (int64_t)s * p.rows]);
    sums[0][threadIdx.x] = most;
    __syncthreads();
    for (int s = 0; s < j.shares; ++s) most = fmaxf(most, sums[0][(int)threadIdx.x + (s - o.share) * j.quads]);
    __syncthreads();
    if (there) {
#pragma unroll 4
        for (int s = o.share; s < p.splits; s += j.shares) {
            const float lse = p.part_lse[at + (int64_t)s * p.rows];
            if (lse == -__builtin_inff() || o.d >= p.dim) continue;         // a part that sees nothing
            const float w = __builtin_amdgcn_exp2f(lse - most);
            float u[4];
            gm_load<float, 4>(u, p.part + (at + (int64_t)s * p.rows) * p.dim + o.d, p.dim - o.d);
            v[4] += w;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = fmaf(w, u[i], v[i]);
        }
    }
    if (!at_join<5>(j, sums, v) || !there || o.d >= p.dim) return;
    const bool none = v[4] == 0.f;
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = none ? 0.f : v[i] / v[4];
    const int64_t to = ((b * p.nq + pos) * p.heads + head) * p.dim + o.d;
    gm_store<E, 4>(y, (E *)p.y + to, p.dim - o.d);
    if (p.rest) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = at_rest<E>(y[i]);
        gm_store<E, 4>(y, (E *)p.rest + to, p.dim - o.d);
    }
    if (p.lse && o.d == 0) p.lse[(b * p.heads + head) * p.nq + pos] = none ? __builtin_inff() : most + __builtin_amdgcn_logf(v[4]);
}

// Sums of parts [splits][n], in a fixed order; dQ's come by head of keys and row.
template <typename E, bool DQ>
__global__ __launch_bounds__(AT_TPB) void attention_sum_kernel(AttentionP p, AtJoin j)
{
    __shared__ float sums[4][AT_TPB];
    const AtJoinPlace o = at_join_place(j);
    int64_t from, step;
    E *to;
    if constexpr (DQ) {
        const int64_t group = o.row / p.rows, b = group / p.kv_heads;
        const int row = (int)(o.row - group * p.rows), pos = row / p.share, head = (int)(group % p.kv_heads) * p.share + row % p.share;
        from = group * p.splits * p.rows + row;
        step = p.rows;
        to = (E *)p.dq + ((b * p.nq + pos) * p.heads + head) * p.dim;
    } else {
        from = o.row;
        step = j.rows;
        to = o.row < j.rows / 2 ? (E *)p.dk + o.row * p.dim : (E *)p.dv + (o.row - j.rows / 2) * p.dim;
    }
    const bool there = o.row < j.rows && o.d < p.dim;
    float v[4] = {};
    if (there) {
#pragma unroll 4
        for (int s = o.share; s < p.splits; s += j.shares) {
            float u[4];
            gm_load<float, 4>(u, p.part + (from + s * step) * p.dim + o.d, p.dim - o.d);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += u[i];
        }
    }
    if (at_join<4>(j, sums, v) && there) gm_store<E, 4>(v, to + o.d, p.dim - o.d);
}

// Rows [batch][n][heads][dim] of any strides and alignment laid out anew, with `wide` components, zeros behind dim.
struct PackP { int64_t rows, sb, sn, sh; int n, heads, dim, wide; const void *from; void *to; };
template <typename E>
__global__ __launch_bounds__(AT_TPB) void attention_pack_kernel(PackP p)
{
    constexpr int V = fe_width<E>;
    const int chunks = p.wide / V;
    const int64_t total = p.rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * AT_TPB + threadIdx.x; i < total; i += (int64_t)gridDim.x * AT_TPB) {
        const int64_t r = i / chunks, head = r % p.heads, pos = r / p.heads % p.n, b = r / p.heads / p.n;
        const int d = (int)(i - r * chunks) * V;
        E v[V];
        gm_load<E, V>(v, (const E *)p.from + b * p.sb + pos * p.sn + head * p.sh + d, p.dim - d);
        gm_store<E, V>(v, (E *)p.to + r * p.wide + d, V);
    }
}

static unsigned at_flat(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + AT_TPB - 1) / AT_TPB, 8192)); }
static int at_units() { const int n = fgnn_current_device_compute_units(); return n > 0 ? n : 256; }
static int at_wide(int dim, int type) { const int v = 16 / fe_size(type); return (dim + v - 1) / v * v; }
// Whether rows do not all start at 16 bytes and hold whole 16 bytes, or lie 2^24 bytes apart or more.
static bool at_loose(const void *p, const int64_t *strides, int dim, int type)
{
    const int64_t size = fe_size(type);
    return (((uintptr_t)p | strides[0] * size | strides[1] * size | strides[2] * size | dim * size) & 15) || strides[1] * size >= 1 << 24;
}
static size_t at_pack_bytes(int64_t batch, int64_t n, int64_t heads, int dim, int type) { return fgnn_align256((size_t)batch * n * heads * at_wide(dim, type) * fe_size(type)); }
static int at_pack(const void *&p, int64_t &sb, int64_t &sn, int64_t &sh, int batch, int n, int heads, int dim, int type, char *&space, hipStream_t st)
{
    PackP k{(int64_t)batch * n * heads, sb, sn, sh, n, heads, dim, at_wide(dim, type), p, space};
    space += at_pack_bytes(batch, n, heads, dim, type);
    p = k.to;
    sh = k.wide;
    sn = (int64_t)heads * sh;
    sb = n * sn;
    if (k.rows == 0) return 0;
    fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((attention_pack_kernel<E>), dim3(at_flat(k.rows * (k.wide / fe_width<E>))), dim3(AT_TPB), 0, st, k); });
    return fgnn_launch_status("attention_pack_kernel");
}

// Rows of parts joined: a share for every four parts, as far as a workgroup's threads go.
static AtJoin at_joined(int64_t rows, int dim, int splits, unsigned &grid)
{
    AtJoin j{1, 1, rows};
    while (j.quads * 4 < dim) j.quads *= 2;
    while (j.shares * 4 < splits && j.quads * j.shares < AT_TPB) j.shares *= 2;
    const int side = AT_TPB / (j.quads * j.shares);
    grid = (unsigned)((rows + side - 1) / side);
    return j;
}

// Waves and tiles of a pass, and the parts that its long side is cut into where there are too few workgroups for the device.
static AtShape at_shape(AttentionP &p, int what, int type)
{
    AtShape s;
    s.dim = p.dim <= 64 ? 64 : p.dim <= 128 ? 128 : 256;
    s.tile = what == AT_DKV ? AT_ROWS_DKV : fe_size(type) == 4 ? 32 : 64;
    // As many waves as the rows fill: one query to 16 x 4096 keys, 8 heads of 64 in fp32, 64 us for 89 with four waves; 64 queries to 232,965 keys in bf16, training, 476 for 514.
    // (fp32 tiles of more than 64 components wait in registers on their way, for which one wave alone has no room: one query to 16 x 4096 keys of 128 components 698 us for 219.)
    s.waves = what == AT_DKV || p.rows > 64 || (fe_size(type) == 4 && s.dim > 64) ? 4 : p.rows > 32 ? 2 : 1;
    if (s.waves < 4) s.tile = 32;
    const int64_t columns = what == AT_DKV ? p.nk : p.rows, walked = what == AT_DKV ? (int64_t)((p.nq + s.tile - 1) / s.tile) * p.share : (p.nk + s.tile - 1) / s.tile;
    p.tiles = (int)((columns + 32 * s.waves - 1) / (32 * s.waves));
    const int64_t groups = std::max<int64_t>(1, (int64_t)p.tiles * p.kv_heads * p.batch), wanted = (int64_t)at_units() * 8 / s.waves;
    const int64_t most = std::max<int64_t>(1, walked / 4);
    p.splits = (int)std::min<int64_t>({std::max<int64_t>(1, wanted / groups), most, 256});
    p.per = (int)((walked + p.splits - 1) / p.splits);
    p.splits = p.per ? (int)((walked + p.per - 1) / p.per) : 1;
    if (p.splits < 1) p.splits = 1;
    return s;
}
static size_t at_part_bytes(const AttentionP &p, int what)
{
    if (p.splits < 2) return 0;
    if (what == AT_DKV) return fgnn_align256((size_t)p.splits * 2 * p.batch * p.nk * p.kv_heads * p.dim * sizeof(float));
    return fgnn_align256((size_t)p.batch * p.kv_heads * p.splits * p.rows * (p.dim + 1) * sizeof(float));
}
static int64_t at_grid(const AttentionP &p) { return (int64_t)p.tiles * p.splits * p.kv_heads * p.batch; }

static bool at_limits(int nq, int nk, int share) { return (int64_t)nq * share < 1LL << 31 && nk < (1LL << 31) - 128 && nq < (1LL << 31) - 128; }
static int at_check(const char *who, int batch, int nq, int nk, int heads, int kv_heads, int dim, int type)
{
    FGNN_REQUIRE(batch >= 0 && nq >= 0 && nk >= 0 && kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0 && dim >= 1, FGNN_ERR_SHAPE,
                 "%s: bad sizes batch=%d queries=%d keys=%d heads=%d kv_heads=%d dim=%d", who, batch, nq, nk, heads, kv_heads, dim);
    FGNN_REQUIRE(fe_is_float(type), FGNN_ERR_SHAPE, "%s: element type %d", who, type);
    FGNN_REQUIRE(dim <= 256, FGNN_ERR_LIMIT, "%s: heads of %d components, more than 256", who, dim);
    FGNN_REQUIRE(at_limits(nq, nk, heads / kv_heads), FGNN_ERR_LIMIT, "%s: queries=%d keys=%d", who, nq, nk);
    return 0;
}
// (offsets inside a tile are unsigned)
static bool at_negative(const int64_t *strides, int n) { return std::any_of(strides, strides + n, [](int64_t s) { return s < 0; }); }
static AttentionP at_problem(int batch, int nq, int nk, int heads, int kv_heads, int dim)
{
    AttentionP p = {};
    p.batch = batch; p.nq = nq; p.nk = nk; p.heads = heads; p.kv_heads = kv_heads; p.dim = dim;
    p.share = heads / kv_heads;
    p.rows = nq * p.share;
    // row / share by a multiplication (for rows below 2^31)
    while ((1LL << p.share_shift) < p.share) ++p.share_shift;
    p.share_mul = (uint32_t)(((1ULL << 32) * ((1ULL << p.share_shift) - p.share)) / p.share + 1);
    return p;
}
// Whether a pass can be launched: a launch has fewer than 2^32 threads.
static int at_fits(int what, const AtShape &s, const AttentionP &p)
{
    const int64_t grid = at_grid(p), joined = p.splits < 2 ? 0 : (int64_t)p.batch * p.kv_heads * (what == AT_DKV ? 2LL * p.nk : p.rows);
    FGNN_REQUIRE(grid * s.waves < 1LL << 26 && joined < 1LL << 24, FGNN_ERR_LIMIT, "attention: %lld workgroups of %d waves", (long long)grid, s.waves);
    return 0;
}
static int at_run(int what, int type, const AtShape &s, const AttentionP &p, hipStream_t st)
{
    const int64_t grid = at_grid(p);
    if (grid == 0) return 0;
    if (const int rc = at_fits(what, s, p)) return rc;
    fe_dispatch(type, [&]<typename E>() { at_launch<E>(what, s, p, (unsigned)grid, st); });
    return fgnn_launch_status(what == AT_FORWARD ? "attention_kernel" : what == AT_DQ ? "attention_dq_kernel" : "attention_dkv_kernel");
}
// The backward pass's limits, which are looked at before its first launch, and by a caller before a forward pass that trains: the pass of dK and dV has four waves for
// every sample and head of keys, however few keys there are.
extern "C" int fgnn_attention_backward_check(int batch, int nq, int nk, int heads, int kv_heads, int dim, int type, int dq, int dkv)
{
    int rc = at_check("fgnn_attention_backward", batch, nq, nk, heads, kv_heads, dim, type);
    if (rc || batch == 0) return rc;
    AttentionP p = at_problem(batch, nq, nk, heads, kv_heads, dim);
    for (const int what : {AT_DQ, AT_DKV}) {
        if (what == AT_DQ ? !dq || nq == 0 : !dkv || nk == 0) continue;
        const AtShape s = at_shape(p, what, type);
        if ((rc = at_fits(what, s, p))) return rc;
    }
    return 0;
}

extern "C" size_t fgnn_attention_workspace_bytes(int batch, int nq, int nk, int heads, int kv_heads, int dim, int type, const void *k, const void *v, const int64_t *strides)
{
    if (batch < 1 || nq < 1 || nk < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 1 || dim > 256 || !at_limits(nq, nk, heads / kv_heads) || !fe_is_float(type) || !strides) return 0;
    AttentionP p = at_problem(batch, nq, nk, heads, kv_heads, dim);
    at_shape(p, AT_FORWARD, type);
    const size_t pack = at_pack_bytes(batch, nk, kv_heads, dim, type);
    return (at_loose(k, strides + 3, dim, type) ? pack : 0) + (at_loose(v, strides + 6, dim, type) ? pack : 0) + at_part_bytes(p, AT_FORWARD);
}

extern "C" int fgnn_attention_kept(int batch, int nq, int nk, int heads, int kv_heads, int dim, int type, const void *q, const void *k, const void *v, const int64_t *strides,
                                   const void *lengths, int wide, const uint8_t *mask, float scale, void *y, void *rest, float *lse, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = at_check("fgnn_attention", batch, nq, nk, heads, kv_heads, dim, type);
    if (rc || batch == 0 || nq == 0) return rc;
    FGNN_REQUIRE(scale > 0.f && scale < __builtin_inff(), FGNN_ERR_SHAPE, "fgnn_attention: scale %g", (double)scale);
    FGNN_REQUIRE(q && y && strides && (nk == 0 || (k && v)), FGNN_ERR_NULL, "fgnn_attention: NULL argument");
    FGNN_REQUIRE(!at_negative(strides, 9), FGNN_ERR_SHAPE, "fgnn_attention: negative strides");
    const size_t bytes = fgnn_attention_workspace_bytes(batch, nq, nk, heads, kv_heads, dim, type, k, v, strides);
    FGNN_REQUIRE(bytes == 0 || (workspace && workspace_bytes >= bytes), FGNN_ERR_WORKSPACE, "fgnn_attention: workspace of %zu bytes", workspace_bytes);
    hipStream_t st = (hipStream_t)stream;
    AttentionP p = at_problem(batch, nq, nk, heads, kv_heads, dim);
    p.q = q; p.k = k; p.v = v;
    p.qb = strides[0]; p.qn = strides[1]; p.qh = strides[2]; p.kb = strides[3]; p.kn = strides[4]; p.kh = strides[5]; p.vb = strides[6]; p.vn = strides[7]; p.vh = strides[8];
    p.lengths = lengths; p.wide = wide; p.mask = mask;
    p.scale = scale; p.log2_scale = scale * 1.44269504f;
    p.y = y; p.lse = lse; p.rest = fe_size(type) == 2 ? rest : nullptr;
    char *space = (char *)workspace;
    if (nk && at_loose(k, strides + 3, dim, type) && (rc = at_pack(p.k, p.kb, p.kn, p.kh, batch, nk, kv_heads, dim, type, space, st))) return rc;
    if (nk && at_loose(v, strides + 6, dim, type) && (rc = at_pack(p.v, p.vb, p.vn, p.vh, batch, nk, kv_heads, dim, type, space, st))) return rc;
    const AtShape s = at_shape(p, AT_FORWARD, type);
    p.part = (float *)space;
    p.part_lse = p.part + (size_t)batch * kv_heads * p.splits * p.rows * dim;
    if ((rc = at_run(AT_FORWARD, type, s, p, st)) || p.splits < 2) return rc;
    unsigned grid;
    const AtJoin j = at_joined((int64_t)batch * nq * heads, dim, p.splits, grid);
    fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((attention_join_kernel<E>), dim3(grid), dim3(AT_TPB), 0, st, p, j); });
    return fgnn_launch_status("attention_join_kernel");
}

extern "C" int fgnn_attention(int batch, int nq, int nk, int heads, int kv_heads, int dim, int type, const void *q, const void *k, const void *v, const int64_t *strides,
                              const void *lengths, int wide, const uint8_t *mask, float scale, void *y, float *lse, void *workspace, size_t workspace_bytes, void *stream)
{
    return fgnn_attention_kept(batch, nq, nk, heads, kv_heads, dim, type, q, k, v, strides, lengths, wide, mask, scale, y, nullptr, lse, workspace, workspace_bytes, stream);
}

extern "C" size_t fgnn_attention_backward_workspace_bytes(int batch, int nq, int nk, int heads, int kv_heads, int dim, int type, const void *q, const void *k, const void *v, const void *g,
                                                          const int64_t *strides)
{
    if (batch < 1 || nq < 1 || nk < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || dim < 1 || dim > 256 || !at_limits(nq, nk, heads / kv_heads) || !fe_is_float(type) || !strides) return 0;
    AttentionP p = at_problem(batch, nq, nk, heads, kv_heads, dim);
    at_shape(p, AT_DQ, type);
    size_t part = at_part_bytes(p, AT_DQ);
    at_shape(p, AT_DKV, type);
    part = std::max(part, at_part_bytes(p, AT_DKV));
    const size_t keys = at_pack_bytes(batch, nk, kv_heads, dim, type), queries = at_pack_bytes(batch, nq, heads, dim, type);
    return fgnn_align256((size_t)batch * heads * nq * sizeof(float)) + part + (at_loose(q, strides, dim, type) ? queries : 0) + (at_loose(k, strides + 3, dim, type) ? keys : 0) +
           (at_loose(v, strides + 6, dim, type) ? keys : 0) + (at_loose(g, strides + 9, dim, type) ? queries : 0);
}

extern "C" int fgnn_attention_kept_backward(int batch, int nq, int nk, int heads, int kv_heads, int dim, int type, const void *q, const void *k, const void *v, const void *y,
                                            const void *rest, const void *g, const int64_t *strides, const void *lengths, int wide, const uint8_t *mask, float scale, const float *lse, void *dq,
                                            void *dk, void *dv, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = fgnn_attention_backward_check(batch, nq, nk, heads, kv_heads, dim, type, dq != nullptr, dk != nullptr);
    if (rc || batch == 0) return rc;
    FGNN_REQUIRE(scale > 0.f && scale < __builtin_inff(), FGNN_ERR_SHAPE, "fgnn_attention_backward: scale %g", (double)scale);
    FGNN_REQUIRE((dk == nullptr) == (dv == nullptr), FGNN_ERR_NULL, "fgnn_attention_backward: dk and dv are formed together");
    FGNN_REQUIRE(strides && (nq == 0 || (q && y && g && lse)) && (nk == 0 || (k && v)), FGNN_ERR_NULL, "fgnn_attention_backward: NULL argument");
    FGNN_REQUIRE(!at_negative(strides, 12), FGNN_ERR_SHAPE, "fgnn_attention_backward: negative strides");
    const size_t bytes = fgnn_attention_backward_workspace_bytes(batch, nq, nk, heads, kv_heads, dim, type, q, k, v, g, strides);
    FGNN_REQUIRE(bytes == 0 || (workspace && workspace_bytes >= bytes), FGNN_ERR_WORKSPACE, "fgnn_attention_backward: workspace of %zu bytes", workspace_bytes);
    hipStream_t st = (hipStream_t)stream;
    AttentionP p = at_problem(batch, nq, nk, heads, kv_heads, dim);
    p.q = q; p.k = k; p.v = v; p.g = g;
    p.qb = strides[0]; p.qn = strides[1]; p.qh = strides[2]; p.kb = strides[3]; p.kn = strides[4]; p.kh = strides[5]; p.vb = strides[6]; p.vn = strides[7]; p.vh = strides[8];
    p.gb = strides[9]; p.gn = strides[10]; p.gh = strides[11];
    p.lengths = lengths; p.wide = wide; p.mask = mask;
    p.scale = scale; p.log2_scale = scale * 1.44269504f;
    p.y = const_cast<void *>(y); p.lse = const_cast<float *>(lse); p.rest = fe_size(type) == 2 ? const_cast<void *>(rest) : nullptr;
    p.dq = dq; p.dk = dk; p.dv = dv;
    char *space = (char *)workspace;
    if (nq) {
        p.delta = (float *)space;
        space += fgnn_align256((size_t)batch * heads * nq * sizeof(float));
        if (!dq) {
            fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((attention_delta_kernel<E>), dim3(at_flat(2LL * batch * nq * heads)), dim3(AT_TPB), 0, st, p); });
            if ((rc = fgnn_launch_status("attention_delta_kernel"))) return rc;
        }
        if (at_loose(q, strides, dim, type) && (rc = at_pack(p.q, p.qb, p.qn, p.qh, batch, nq, heads, dim, type, space, st))) return rc;
        if (at_loose(k, strides + 3, dim, type) && (rc = at_pack(p.k, p.kb, p.kn, p.kh, batch, nk, kv_heads, dim, type, space, st))) return rc;
        if (at_loose(v, strides + 6, dim, type) && (rc = at_pack(p.v, p.vb, p.vn, p.vh, batch, nk, kv_heads, dim, type, space, st))) return rc;
        if (at_loose(g, strides + 9, dim, type) && (rc = at_pack(p.g, p.gb, p.gn, p.gh, batch, nq, heads, dim, type, space, st))) return rc;
    }
    p.part = (float *)space;
    unsigned grid;
    if (dq && nq) {
        const AtShape s = at_shape(p, AT_DQ, type);
        if ((rc = at_run(AT_DQ, type, s, p, st))) return rc;
        if (p.splits > 1) {
            const AtJoin j = at_joined((int64_t)batch * nq * heads, dim, p.splits, grid);
            fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((attention_sum_kernel<E, true>), dim3(grid), dim3(AT_TPB), 0, st, p, j); });
            if ((rc = fgnn_launch_status("attention_sum_kernel"))) return rc;
        }
    }
    if (dk && nk) {
        const AtShape s = at_shape(p, AT_DKV, type);
        if ((rc = at_run(AT_DKV, type, s, p, st))) return rc;
        if (p.splits > 1) {
            const AtJoin j = at_joined(2LL * batch * nk * kv_heads, dim, p.splits, grid);
            fe_dispatch(type, [&]<typename E>() { hipLaunchKernelGGL((attention_sum_kernel<E, false>), dim3(grid), dim3(AT_TPB), 0, st, p, j); });
            return fgnn_launch_status("attention_sum_kernel");
        }
    }
    return 0;
}

extern "C" int fgnn_attention_backward(int batch, int nq, int nk, int heads, int kv_heads, int dim, int type, const void *q, const void *k, const void *v, const void *y, const void *g,
                                       const int64_t *strides, const void *lengths, int wide, const uint8_t *mask, float scale, const float *lse, void *dq, void *dk, void *dv, void *workspace,
                                       size_t workspace_bytes, void *stream)
{
    return fgnn_attention_kept_backward(batch, nq, nk, heads, kv_heads, dim, type, q, k, v, y, nullptr, g, strides, lengths, wide, mask, scale, lse, dq, dk, dv, workspace, workspace_bytes,
                                        stream);
}
