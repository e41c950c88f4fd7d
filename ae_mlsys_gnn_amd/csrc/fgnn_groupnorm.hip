// Group norm with an activation over channels-last features x [batch][points][channels]: of every sample and every group of channels
//   m = mean x,   s = (mean (x - m)^2 + eps)^-1/2,   u = (x - m) s,   z = u w_c + b_c,   y = act(z)
// and its gradient.  With d = gy act'(z), and A_c = sum d, B_c = sum d u over a sample's points,
//   dx = s (d w_c - mean_group(w A) - u mean_group(w B)),   dw_c = sum over samples of B_c,   db_c of A_c.
// Bound by memory.  Everything is formed from sums a sample and channel, so that a thread keeps its 16 bytes of channels over many points, a group
// may have any number of channels, and the sums over chunks and channels are added in 64 bits in a fixed order.
#include <algorithm>
#include "fgnn_gemm.h"

#define GN_TPB 256
#define GN_GRID (1 << 20)                   // most workgroups: a launch has fewer than 2^32 threads
struct GroupNormP {
    int64_t batch, points;
    int cols, groups, width;                // width: channels a group
    const void *x; int64_t ldx, sx;         // strides of points and samples, in elements
    const void *w, *b; int wtype, btype;    // NULL: ones, zeros
    float eps, slope; int act;
    void *y;
    float *mean, *rstd;                     // [batch][groups]
    const void *gy; void *dx;               // contiguous
    int chunks; int64_t rows;               // parts of a sample's points, and points of each
    int tiles, lanes;                       // parts of the channels, and vectors of each
    float *part;                            // [batch][chunks][2][cols]
    float *sums, *group;                    // backward: [batch][2][cols] A and B, [batch][groups][2] means
};

template <typename E, int V>
__device__ __forceinline__ void gn_load(float (&v)[V], const E *row, int left)
{
    gm_load<E, V>(v, row, left);
}
// The statistics, weights and bias of a thread's V channels.
template <int V> struct GnCols { float mean[V], rstd[V], w[V], b[V]; };
template <int V>
__device__ __forceinline__ void gn_columns(const GroupNormP &p, int64_t sample, int c, GnCols<V> &o)
{
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int j = min(c + i, p.cols - 1);
        const int64_t g = sample * p.groups + j / p.width;
        o.mean[i] = p.mean[g];
        o.rstd[i] = p.rstd[g];
        o.w[i] = p.w ? fe_load(p.w, j, p.wtype) : 1.f;
        o.b[i] = p.b ? fe_load(p.b, j, p.btype) : 0.f;
    }
}
// d and u of V elements, from x and gy
template <int V>
__device__ __forceinline__ void gn_slope(const GroupNormP &p, const GnCols<V> &o, float (&x)[V], float (&g)[V])
{
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        x[i] = (x[i] - o.mean[i]) * o.rstd[i];
        z[i] = fmaf(x[i], o.w[i], o.b[i]);
    }
    gm_act_slope(g, z, p.act, p.slope);
}

// A workgroup's place: sample, chunk of points, tile of channels.
struct GnPlace { int64_t sample, first, last; int chunk, c, left, row, step; bool on; };
template <int V>
__device__ __forceinline__ GnPlace gn_place(const GroupNormP &p, int64_t item)
{
    GnPlace o;
    const int tile = (int)(item % p.tiles);
    item /= p.tiles;
    o.chunk = (int)(item % p.chunks);
    o.sample = item / p.chunks;
    o.first = o.chunk * p.rows;
    o.last = min(p.points, o.first + p.rows);
    o.step = GN_TPB / p.lanes;
    o.row = (int)threadIdx.x / p.lanes;
    o.c = (tile * p.lanes + (int)threadIdx.x % p.lanes) * V;
    o.left = p.cols - o.c;
    o.on = o.row < o.step && o.left > 0;
    return o;
}

// Sums over a chunk of points, a channel each: of x - k and its square, with k the channel's first value in the sample (squares of what is far from 0
// would lose the variance), or of d and d u.
template <typename E, bool BACKWARD>
__global__ __launch_bounds__(GN_TPB) void gn_sums_kernel(GroupNormP p)
{
    constexpr int V = fe_width<E>, U = BACKWARD ? 2 : 4;
    __shared__ float red[2][GN_TPB * V];
    const int64_t items = p.batch * p.chunks * p.tiles;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const GnPlace o = gn_place<V>(p, item);
        float a[V], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = b[i] = 0.f;
        if (o.on) {
            const E *x = (const E *)p.x + o.sample * p.sx + o.c;
            const E *gy = BACKWARD ? (const E *)p.gy + o.sample * p.points * p.cols + o.c : nullptr;
            float k[V];
            GnCols<V> cols;
            if constexpr (BACKWARD) gn_columns<V>(p, o.sample, o.c, cols);
            else gn_load<E, V>(k, x, o.left);
            auto add = [&](float (&v)[V], float (&g)[V]) {
                if constexpr (BACKWARD) {
                    gn_slope<V>(p, cols, v, g);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        a[i] += g[i];
                        b[i] = fmaf(g[i], v[i], b[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float t = v[i] - k[i];
                        a[i] += t;
                        b[i] = fmaf(t, t, b[i]);
                    }
                }
            };
            int64_t r = o.first + o.row;
            for (; r + (U - 1) * o.step < o.last; r += U * o.step) {
                float v[U][V], g[U][V];
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    gn_load<E, V>(v[j], x + (r + j * o.step) * p.ldx, o.left);
                    if constexpr (BACKWARD) gn_load<E, V>(g[j], gy + (r + j * o.step) * p.cols, o.left);
                }
#pragma unroll
                for (int j = 0; j < U; ++j) add(v[j], g[j]);
            }
            for (; r < o.last; r += o.step) {
                float v[V], g[V];
                gn_load<E, V>(v, x + r * p.ldx, o.left);
                if constexpr (BACKWARD) gn_load<E, V>(g, gy + r * p.cols, o.left);
                add(v, g);
            }
        }
        __syncthreads();                    // the sums before are read
#pragma unroll
        for (int i = 0; i < V; ++i) {
            red[0][threadIdx.x * V + i] = a[i];
            red[1][threadIdx.x * V + i] = b[i];
        }
        __syncthreads();
        const int tile0 = o.c - (int)(threadIdx.x % p.lanes) * V, n = min(p.lanes * V, p.cols - tile0);
        for (int t = threadIdx.x; t < 2 * n; t += GN_TPB) {
            const int which = t >= n, c = t - which * n;
            float v = 0.f;
            for (int i = 0; i < o.step; ++i) v += red[which][i * p.lanes * V + c];
            p.part[((o.sample * p.chunks + o.chunk) * 2 + which) * p.cols + tile0 + c] = v;
        }
    }
}

// The sum of v over the workgroup's threads, in a fixed order; every thread gets it.  red: one value a wave.
template <int N>
__device__ __forceinline__ void gn_all(double (&v)[N], double (*red)[N])
{
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) v[j] += __shfl_xor(v[j], o, 64);
    __syncthreads();
    if (fg_lane() == 0)
#pragma unroll
        for (int j = 0; j < N; ++j) red[threadIdx.x >> 6][j] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (red[0][j] + red[1][j]) + (red[2][j] + red[3][j]);
}

// Statistics of a sample's group from the sums about the channels' first values k: with k0 the group's first of all, sum (x - k0)^2 = sum over
// channels of s2 + 2 (k - k0) s1 + points (k - k0)^2.
template <typename E>
__global__ __launch_bounds__(GN_TPB) void gn_stats_kernel(GroupNormP p)
{
    __shared__ double red[GN_TPB / 64][2];
    const int64_t items = p.batch * p.groups;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t sample = item / p.groups;
        const int c0 = (int)(item % p.groups) * p.width;
        const E *x = (const E *)p.x + sample * p.sx + c0;
        const double k0 = (double)(float)x[0];
        double v[2] = {0., 0.};
        const int64_t n = (int64_t)p.chunks * p.width;
        for (int64_t i = threadIdx.x; i < n; i += GN_TPB) {
            const int64_t chunk = i / p.width;
            const int c = (int)(i % p.width);
            const float *part = p.part + ((sample * p.chunks + chunk) * 2) * p.cols + c0 + c;
            const double s1 = part[0], s2 = part[p.cols], k = (double)(float)x[c] - k0;
            const double rows = (double)(min(p.points, (chunk + 1) * p.rows) - chunk * p.rows);
            v[0] += s1 + rows * k;
            v[1] += s2 + k * (2. * s1 + rows * k);
        }
        gn_all<2>(v, red);
        if (threadIdx.x == 0) {
            const double count = (double)p.points * p.width, mean = v[0] / count, var = v[1] / count - mean * mean;
            p.mean[item] = (float)(k0 + mean);
            p.rstd[item] = (float)(1. / sqrt((var > 0. || var != var ? var : 0.) + (double)p.eps));
        }
    }
}

// The sums of A and B over the chunks, and of w A and w B over a group.
__global__ __launch_bounds__(GN_TPB) void gn_group_kernel(GroupNormP p)
{
    __shared__ double red[GN_TPB / 64][2], col[2][GN_TPB];
    const int64_t items = p.batch * p.groups;
    const int C = min(p.width, GN_TPB), Q = GN_TPB / C, q = (int)threadIdx.x / C, lane = (int)threadIdx.x % C;      // channels at a time, threads of each
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t sample = item / p.groups;
        const int c0 = (int)(item % p.groups) * p.width;
        double v[2] = {0., 0.};
        for (int first = 0; first < p.width; first += C) {
            const int c = c0 + first + lane;
            const bool on = q < Q && first + lane < p.width;
            double a[2] = {0., 0.};
            if (on)
                for (int i = q; i < p.chunks; i += Q) {
                    const float *part = p.part + ((sample * p.chunks + i) * 2) * p.cols + c;
                    a[0] += part[0];
                    a[1] += part[p.cols];
                }
            __syncthreads();
            col[0][threadIdx.x] = a[0];
            col[1][threadIdx.x] = a[1];
            __syncthreads();
            if (on && q == 0) {
                for (int i = 1; i < Q; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) a[j] += col[j][i * C + lane];
                const double w = p.w ? fe_load(p.w, c, p.wtype) : 1.f;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    p.sums[(sample * 2 + j) * p.cols + c] = (float)a[j];
                    v[j] += w * a[j];
                }
            }
        }
        gn_all<2>(v, red);
        if (threadIdx.x < 2) p.group[item * 2 + threadIdx.x] = (float)((threadIdx.x ? v[1] : v[0]) / ((double)p.points * p.width));
    }
}

// y, or dx, of a chunk of points.
template <typename E, bool BACKWARD>
__global__ __launch_bounds__(GN_TPB) void gn_apply_kernel(GroupNormP p)
{
    constexpr int V = fe_width<E>, U = BACKWARD ? 2 : 4;
    const int64_t items = p.batch * p.chunks * p.tiles;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const GnPlace o = gn_place<V>(p, item);
        if (!o.on) continue;
        const E *x = (const E *)p.x + o.sample * p.sx + o.c;
        const int64_t base = o.sample * p.points * p.cols + o.c;
        GnCols<V> cols;
        gn_columns<V>(p, o.sample, o.c, cols);
        float ma[V], mb[V];
        if constexpr (BACKWARD) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int64_t g = o.sample * p.groups + min(o.c + i, p.cols - 1) / p.width;
                ma[i] = p.group[2 * g];
                mb[i] = p.group[2 * g + 1];
            }
        }
        auto finish = [&](float (&v)[V], float (&g)[V], int64_t r) {
            if constexpr (BACKWARD) {
                gn_slope<V>(p, cols, v, g);
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = cols.rstd[i] * (fmaf(g[i], cols.w[i], -ma[i]) - v[i] * mb[i]);
                gm_store<E, V>(g, (E *)p.dx + base + r * p.cols, o.left);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = fmaf((v[i] - cols.mean[i]) * cols.rstd[i], cols.w[i], cols.b[i]);
                gm_act(v, p.act, p.slope);
                gm_store<E, V>(v, (E *)p.y + base + r * p.cols, o.left);
            }
        };
        int64_t r = o.first + o.row;
        for (; r + (U - 1) * o.step < o.last; r += U * o.step) {
            float v[U][V], g[U][V];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                gn_load<E, V>(v[j], x + (r + j * o.step) * p.ldx, o.left);
                if constexpr (BACKWARD) gn_load<E, V>(g[j], (const E *)p.gy + base + (r + j * o.step) * p.cols, o.left);
            }
#pragma unroll
            for (int j = 0; j < U; ++j) finish(v[j], g[j], r + j * o.step);
        }
        for (; r < o.last; r += o.step) {
            float v[V], g[V];
            gn_load<E, V>(v, x + r * p.ldx, o.left);
            if constexpr (BACKWARD) gn_load<E, V>(g, (const E *)p.gy + base + r * p.cols, o.left);
            finish(v, g, r);
        }
    }
}

// dw and db: the sums [rows][2][cols] over the rows, 16 channels a workgroup at a time, 64 rows side by side, in 64 bits.
__global__ __launch_bounds__(1024) void gn_weights_kernel(const float *__restrict__ sums, int64_t rows, int cols, void *dw, int wtype, void *db, int btype)
{
    __shared__ double red[64][17];
    const int c = (int)threadIdx.x & 15, q = (int)threadIdx.x >> 4;
    const int tiles = (cols + 15) / 16;
    for (int64_t item = blockIdx.x; item < 2 * (int64_t)tiles; item += gridDim.x) {
        const int which = (int)(item / tiles), col = (int)(item % tiles) * 16 + c;          // 0: A, 1: B
        double v = 0.;
        if (col < cols) {
#pragma unroll 4
            for (int64_t i = q; i < rows; i += 64) v += sums[(2 * i + which) * cols + col];
        }
        __syncthreads();
        red[q][c] = v;
        __syncthreads();
        if (q == 0 && col < cols) {
            for (int i = 1; i < 64; ++i) v += red[i][c];
            if (which && dw) fe_store(dw, col, wtype, (float)v);
            if (!which && db) fe_store(db, col, btype, (float)v);
        }
    }
}

// Chunks of a sample's points and tiles of its channels: about eight workgroups a compute unit, but at least eight points a thread.
static void gn_cut(GroupNormP &p, int type)
{
    const int v = 16 / fe_size(type), vectors = (p.cols + v - 1) / v, cus = fgnn_current_device_compute_units();
    p.width = p.cols / p.groups;
    p.tiles = (vectors + GN_TPB - 1) / GN_TPB;
    p.lanes = (vectors + p.tiles - 1) / p.tiles;
    const int64_t step = GN_TPB / p.lanes, wanted = std::max<int64_t>(1, (int64_t)(cus > 0 ? cus : 256) * 8 / std::max<int64_t>(1, p.batch * p.tiles));
    p.rows = std::max<int64_t>({(p.points + wanted - 1) / wanted, 8 * step, 1});
    p.chunks = (int)((p.points + p.rows - 1) / p.rows);
}
static unsigned gn_grid(int64_t items) { return (unsigned)std::min<int64_t>(items, GN_GRID); }

static int gn_check(const char *who, int64_t batch, int64_t points, int cols, int groups, int type, const void *x, int64_t ldx, int64_t sx, const void *w, int wtype, const void *b,
                    int btype, int act)
{
    FGNN_REQUIRE(batch >= 0 && points >= 0 && cols >= 1 && groups >= 1 && cols % groups == 0 && ldx >= cols && sx >= 0, FGNN_ERR_SHAPE,
                 "%s: bad sizes batch=%lld points=%lld cols=%d groups=%d ldx=%lld", who, (long long)batch, (long long)points, cols, groups, (long long)ldx);
    FGNN_REQUIRE(fe_is_float(type) && (!w || wtype == type || wtype == FGNN_F32) && (!b || btype == type || btype == FGNN_F32), FGNN_ERR_SHAPE,
                 "%s: element type %d with weights of type %d, bias of type %d", who, type, wtype, btype);
    FGNN_REQUIRE(act >= GM_NONE && act <= GM_LEAKY, FGNN_ERR_SHAPE, "%s: activation %d", who, act);
    FGNN_REQUIRE(cols <= 1 << 30 && points <= 1LL << 40 && batch <= (1LL << 31), FGNN_ERR_LIMIT, "%s: batch=%lld points=%lld cols=%d", who, (long long)batch, (long long)points, cols);
    FGNN_REQUIRE(batch == 0 || points == 0 || x, FGNN_ERR_NULL, "%s: NULL argument", who);
    return 0;
}

// The sums of the chunks, then (backward) those of a sample and of a group.
static size_t gn_part_bytes(const GroupNormP &p) { return fgnn_align256((size_t)p.batch * p.chunks * 2 * p.cols * sizeof(float)); }
static size_t gn_sums_bytes(const GroupNormP &p) { return fgnn_align256((size_t)p.batch * 2 * p.cols * sizeof(float)); }
static size_t gn_workspace(int64_t batch, int64_t points, int cols, int groups, int type, int backward)
{
    if (batch < 1 || points < 1 || cols < 1 || groups < 1 || !fe_is_float(type)) return 0;
    GroupNormP p = {};
    p.batch = batch; p.points = points; p.cols = cols; p.groups = groups;
    gn_cut(p, type);
    return gn_part_bytes(p) + (backward ? gn_sums_bytes(p) + fgnn_align256((size_t)batch * groups * 2 * sizeof(float)) : 0);
}
extern "C" size_t fgnn_group_norm_workspace_bytes(int64_t batch, int64_t points, int cols, int groups, int type) { return gn_workspace(batch, points, cols, groups, type, 0); }
extern "C" size_t fgnn_group_norm_backward_workspace_bytes(int64_t batch, int64_t points, int cols, int groups, int type) { return gn_workspace(batch, points, cols, groups, type, 1); }

extern "C" int fgnn_group_norm(int64_t batch, int64_t points, int cols, int groups, int type, const void *x, int64_t ldx, int64_t sx, const void *weight, int wtype, const void *bias,
                               int btype, float eps, int act, float slope, void *y, float *mean, float *rstd, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = gn_check("fgnn_group_norm", batch, points, cols, groups, type, x, ldx, sx, weight, wtype, bias, btype, act);
    if (rc) return rc;
    if (batch == 0 || points == 0) return 0;
    FGNN_REQUIRE(y && mean && rstd, FGNN_ERR_NULL, "fgnn_group_norm: NULL argument");
    GroupNormP p = {batch, points, cols, groups, 0, x, ldx, sx, weight, bias, wtype, btype, eps, slope, act, y, mean, rstd};
    gn_cut(p, type);
    FGNN_REQUIRE(workspace && workspace_bytes >= gn_workspace(batch, points, cols, groups, type, 0), FGNN_ERR_WORKSPACE, "fgnn_group_norm: workspace of %zu bytes", workspace_bytes);
    hipStream_t st = (hipStream_t)stream;
    p.part = (float *)workspace;
    const unsigned grid = gn_grid(batch * p.chunks * p.tiles);
    fe_dispatch(type, [&]<typename E>() {
        hipLaunchKernelGGL((gn_sums_kernel<E, false>), dim3(grid), dim3(GN_TPB), 0, st, p);
        hipLaunchKernelGGL((gn_stats_kernel<E>), dim3(gn_grid(batch * groups)), dim3(GN_TPB), 0, st, p);
        hipLaunchKernelGGL((gn_apply_kernel<E, false>), dim3(grid), dim3(GN_TPB), 0, st, p);
    });
    return fgnn_launch_status("gn_apply_kernel");
}

extern "C" int fgnn_group_norm_backward(int64_t batch, int64_t points, int cols, int groups, int type, const void *gy, const void *x, int64_t ldx, int64_t sx, const void *weight,
                                        int wtype, const void *bias, int btype, int act, float slope, const float *mean, const float *rstd, void *dx, void *dweight, void *dbias,
                                        void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = gn_check("fgnn_group_norm_backward", batch, points, cols, groups, type, x, ldx, sx, weight, wtype, bias, btype, act);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    const bool empty = batch == 0 || points == 0;
    GroupNormP p = {batch, points, cols, groups, 0, x, ldx, sx, weight, bias, wtype, btype, 0.f, slope, act, nullptr, const_cast<float *>(mean), const_cast<float *>(rstd), gy, dx};
    if (!weight) p.wtype = type;
    if (!bias) p.btype = type;
    if (!empty) {
        FGNN_REQUIRE(gy && mean && rstd, FGNN_ERR_NULL, "fgnn_group_norm_backward: NULL argument");
        FGNN_REQUIRE(workspace && workspace_bytes >= gn_workspace(batch, points, cols, groups, type, 1), FGNN_ERR_WORKSPACE, "fgnn_group_norm_backward: workspace of %zu bytes",
                     workspace_bytes);
        gn_cut(p, type);
        p.part = (float *)workspace;
        p.sums = (float *)((char *)workspace + gn_part_bytes(p));
        p.group = (float *)((char *)p.sums + gn_sums_bytes(p));
        const unsigned grid = gn_grid(batch * p.chunks * p.tiles);
        fe_dispatch(type, [&]<typename E>() {
            hipLaunchKernelGGL((gn_sums_kernel<E, true>), dim3(grid), dim3(GN_TPB), 0, st, p);
            hipLaunchKernelGGL(gn_group_kernel, dim3(gn_grid(batch * groups)), dim3(GN_TPB), 0, st, p);
            if (dx) hipLaunchKernelGGL((gn_apply_kernel<E, true>), dim3(grid), dim3(GN_TPB), 0, st, p);
        });
        const int launched = fgnn_launch_status("gn_apply_kernel");
        if (launched) return launched;
    }
    if (dweight || dbias) {
        hipLaunchKernelGGL(gn_weights_kernel, dim3(gn_grid(2 * (((int64_t)cols + 15) / 16))), dim3(1024), 0, st, p.sums, empty ? 0 : batch, cols, dweight, p.wtype, dbias, p.btype);
        return fgnn_launch_status("gn_weights_kernel");
    }
    return 0;
}
