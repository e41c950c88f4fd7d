// Group norm with an activation over channels-last features x [batch][points][channels]: of every sample and every group of channels
//   m = mean x,   s = (mean (x - m)^2 + eps)^-1/2,   u = (x - m) s,   z = u w_c + b_c,   y = act(z)
// and its gradient.  With d = gy act'(z), and A_c = sum d, B_c = sum d u over a sample's points,
//   dx = s (d w_c - mean_group(w A) - u mean_group(w B)),   dw_c = sum over samples of B_c,   db_c of A_c.
// Bound by memory.  A thread keeps its 16 bytes of channels over many points, a group may have any number of channels, and every sum has a fixed order.
// Samples that fit a workgroup's registers are read once: their points' and channels' sums are 32 bits, of the deviations from the mean in a second walk over the registers, and
// what a place adds up for dw and db over its samples is 32 bits too.  Longer samples go in chunks: moments, A and B of a chunk and channel are 32 bits, and are joined over chunks
// and channels in 64.  The places' (samples') parts of dw and db are added in 64 bits on either way.
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

// Vectors that would end behind the last channel begin earlier, where the workgroup's channels leave room: the channels that they share with the vector before are summed there alone,
// and written twice, the same values (element by element 13 x 1433 x 602 fp16 in groups of 43 took 46 us forward and 86 backward, this way 33 and 65).
struct GnVector { int c, shared, left; };   // first channel, how many of them are the vector's before, channels from the first on
template <int V>
__device__ __forceinline__ GnVector gn_vector(int c, int end, int first)
{
    const int from = max(min(c, end - V), first);
    return {from, c - from, end - from};
}
template <typename E>
__device__ __forceinline__ typename fe_vec<E>::type gn_read(const E *p, int left)
{
    typedef typename fe_vec<E>::type vec;
    if (left >= fe_width<E>) return *reinterpret_cast<const vec *>(p);
    vec v = {};
#pragma unroll
    for (int i = 0; i < fe_width<E>; ++i) if (i < left) v[i] = p[i];
    return v;
}
template <typename E, int V>
__device__ __forceinline__ void gn_floats(float (&v)[V], typename fe_vec<E>::type u)
{
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)u[i];
}
// The statistics, weights and bias of a thread's V channels; mean: -mean rstd, so that u = x rstd + mean in one operation, which is off by a rounding of the mean in
// deviations, as the mean itself is.
template <int V> struct GnCols { float mean[V], rstd[V], w[V], b[V]; };
// d and u of V elements, from x and gy.
template <int V>
__device__ __forceinline__ void gn_slope(const GroupNormP &p, const GnCols<V> &o, float (&x)[V], float (&g)[V])
{
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        x[i] = fmaf(x[i], o.rstd[i], o.mean[i]);
        z[i] = fmaf(x[i], o.w[i], o.b[i]);
    }
    gm_act_slope(g, z, p.act, p.slope);
}

// A workgroup's place: sample, chunk of points, tile of channels.
struct GnPlace { int64_t sample, first, last; int chunk, tile0, c, shared, left, row, step; bool on; };
template <int V>
__device__ __forceinline__ GnPlace gn_place(const GroupNormP &p, uint32_t item)
{
    GnPlace o;
    const int tile = (int)(item % (uint32_t)p.tiles);
    item /= (uint32_t)p.tiles;
    o.chunk = (int)(item % (uint32_t)p.chunks);
    o.sample = item / (uint32_t)p.chunks;
    o.first = o.chunk * p.rows;
    o.last = min(p.points, o.first + p.rows);
    o.step = GN_TPB / p.lanes;
    o.row = (int)threadIdx.x / p.lanes;
    o.tile0 = tile * p.lanes * V;
    const int c = o.tile0 + (int)threadIdx.x % p.lanes * V;
    const GnVector v = gn_vector<V>(c, p.cols, o.tile0);
    o.c = v.c;
    o.shared = v.shared;
    o.left = v.left;
    o.on = o.row < o.step && c < p.cols;
    return o;
}

// What a tile's channels are multiplied with and shifted by, formed once a workgroup and handed out through LDS (each thread for its own channels: some thirty loads and eight
// divisions before the first point; 13 x 1433 x 602 fp16: y 19.2 us for 17.8, dx 26.4 for 21.2): z = a x + c with a = rstd w, c = b - mean a; and
//   sums of the backward pass: the mean;      dx = a d + e x + f with e = -rstd^2 mb, f = rstd (mean rstd mb - ma).
enum { GN_VALUES = 2, GN_SUMS = 3, GN_GRADIENT = 4 };
template <int WHAT, int V>
__device__ __forceinline__ void gn_prepare(const GroupNormP &p, const GnPlace &o, float (*co)[GN_TPB * V])
{
    __syncthreads();                        // the ones before are read
    for (int i = threadIdx.x; i < min(p.lanes * V, p.cols - o.tile0); i += GN_TPB) {
        const int j = o.tile0 + i;
        const int64_t g = o.sample * p.groups + j / p.width;
        const float mean = p.mean[g], rstd = p.rstd[g], a = rstd * (p.w ? fe_load(p.w, j, p.wtype) : 1.f);
        co[0][i] = a;
        co[1][i] = fmaf(-mean, a, p.b ? fe_load(p.b, j, p.btype) : 0.f);
        if constexpr (WHAT == GN_SUMS) co[2][i] = mean;
        if constexpr (WHAT == GN_GRADIENT) {
            const float ma = p.group[2 * g], mb = p.group[2 * g + 1];
            co[2][i] = -rstd * rstd * mb;
            co[3][i] = rstd * fmaf(mean * rstd, mb, -ma);
        }
    }
    __syncthreads();
}
template <int V>
__device__ __forceinline__ void gn_take(float (&v)[V], const float *co, const GnPlace &o)
{
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = co[o.c - o.tile0 + (i < o.left ? i : 0)];
}

// Moments of values joined: of n0 with mean m and sum of squared deviations q, and of n1.  Nothing is taken from a value that is larger than the deviations themselves, so an
// outlier, wherever it lies, costs no more than its own rounding (sums of squares about a channel's first value, which were here, lost 1e-3 of the variance where that one was 1000
// deviations off).
template <int V>
__device__ __forceinline__ void gn_join(float &n0, float (&m)[V], float (&q)[V], float n1, const float (&m1)[V], const float (&q1)[V])
{
    const float n = n0 + n1, part = n1 * __builtin_amdgcn_rcpf(n), weight = n0 * part;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float d = m1[i] - m[i];
        m[i] = fmaf(d, part, m[i]);
        q[i] += fmaf(d * weight, d, q1[i]);
    }
    n0 = n;
}
// Means and sums of squared deviations over a chunk of points, a channel each: of four points at a time, joined to a thread's, and the threads' joined pairwise.
template <typename E>
__global__ __launch_bounds__(GN_TPB) void gn_moments_kernel(GroupNormP p)
{
    constexpr int V = fe_width<E>, U = 4;
    typedef typename fe_vec<E>::type vec;
    __shared__ float red[2][GN_TPB][V], counts[GN_TPB];
    const uint32_t items = (uint32_t)(p.batch * p.chunks * p.tiles);
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const GnPlace o = gn_place<V>(p, item);
        const E *x = (const E *)p.x + o.sample * p.sx + o.c;
        float count = 0.f, mean[V], square[V];
#pragma unroll
        for (int i = 0; i < V; ++i) mean[i] = square[i] = 0.f;
        if (o.on) {
            int64_t r = o.first + o.row;
            for (; r + (U - 1) * o.step < o.last; r += U * o.step) {
                vec raw[U];
#pragma unroll
                for (int j = 0; j < U; ++j) raw[j] = gn_read<E>(x + (r + j * o.step) * p.ldx, o.left);
                float v[U][V], m[V], q[V];
#pragma unroll
                for (int j = 0; j < U; ++j) gn_floats<E, V>(v[j], raw[j]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    m[i] = ((v[0][i] + v[1][i]) + (v[2][i] + v[3][i])) * 0.25f;
                    q[i] = 0.f;
#pragma unroll
                    for (int j = 0; j < U; ++j) {
                        const float d = v[j][i] - m[i];
                        q[i] = fmaf(d, d, q[i]);
                    }
                }
                gn_join<V>(count, mean, square, (float)U, m, q);
            }
            for (; r < o.last; r += o.step) {
                float v[V];
                const float none[V] = {};
                gn_floats<E, V>(v, gn_read<E>(x + r * p.ldx, o.left));
                gn_join<V>(count, mean, square, 1.f, v, none);
            }
        }
        // the upper half of the rows to the lower one
        for (int rows = o.step; rows > 1; rows = (rows + 1) / 2) {
            const int half = (rows + 1) / 2;
            __syncthreads();
            if (o.on && o.row >= half && o.row < rows) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    red[0][threadIdx.x][i] = mean[i];
                    red[1][threadIdx.x][i] = square[i];
                }
                counts[threadIdx.x] = count;
            }
            __syncthreads();
            const int other = (int)threadIdx.x + half * p.lanes;
            if (o.on && o.row + half < rows && counts[other] > 0.f) gn_join<V>(count, mean, square, counts[other], red[0][other], red[1][other]);
        }
        if (o.on && o.row == 0) {
            float *part = p.part + (o.sample * p.chunks + o.chunk) * 2 * p.cols + o.c;
            gm_store<float, V>(mean, part, o.left);
            gm_store<float, V>(square, part + p.cols, o.left);
        }
    }
}

// Sums over a chunk of points, a channel each, of d and d (x - mean).
template <typename E, int ACT>
__global__ __launch_bounds__(GN_TPB) void gn_sums_kernel(GroupNormP p)
{
    constexpr int V = fe_width<E>, U = 4;
    typedef typename fe_vec<E>::type vec;
    __shared__ float red[2][GN_TPB * V], co[GN_SUMS][GN_TPB * V];
    const uint32_t items = (uint32_t)(p.batch * p.chunks * p.tiles);
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const GnPlace o = gn_place<V>(p, item);
        const E *x = (const E *)p.x + o.sample * p.sx + o.c;
        const E *gy = (const E *)p.gy + o.sample * p.points * p.cols + o.c;
        float a[V], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) a[i] = b[i] = 0.f;
        gn_prepare<GN_SUMS, V>(p, o, co);
        if (o.on) {
            float mean[V], ca[V], cc[V];
            gn_take<V>(ca, co[0], o);
            gn_take<V>(cc, co[1], o);
            gn_take<V>(mean, co[2], o);
            auto add = [&](vec vx, vec vg) {
                float v[V], z[V], g[V];
                gn_floats<E, V>(v, vx);
                gn_floats<E, V>(g, vg);
#pragma unroll
                for (int i = 0; i < V; ++i) z[i] = fmaf(v[i], ca[i], cc[i]);
                gm_act_slope(g, z, ACT, p.slope);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    a[i] += g[i];
                    b[i] = fmaf(g[i], v[i] - mean[i], b[i]);
                }
            };
            int64_t r = o.first + o.row;
            for (; r + (U - 1) * o.step < o.last; r += U * o.step) {
                vec v[U], g[U];
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    v[j] = gn_read<E>(x + (r + j * o.step) * p.ldx, o.left);
                    g[j] = gn_read<E>(gy + (r + j * o.step) * p.cols, o.left);
                }
#pragma unroll
                for (int j = 0; j < U; ++j) add(v[j], g[j]);
            }
            for (; r < o.last; r += o.step) add(gn_read<E>(x + r * p.ldx, o.left), gn_read<E>(gy + r * p.cols, o.left));
        }
        __syncthreads();                    // the sums before are read
        const int tile0 = o.tile0, n = min(p.lanes * V, p.cols - tile0);
        if (o.on) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i >= o.shared && i < o.left) {
                    red[0][o.row * p.lanes * V + o.c - tile0 + i] = a[i];
                    red[1][o.row * p.lanes * V + o.c - tile0 + i] = b[i];
                }
        }
        __syncthreads();
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

// Statistics of a sample's group from the chunks' and channels' moments, about the first of their means.  Backward: the sums of A and B over the chunks, and the means of w A
// and w B.
template <bool BACKWARD>
__global__ __launch_bounds__(GN_TPB) void gn_group_kernel(GroupNormP p)
{
    __shared__ double red[GN_TPB / 64][2], col[BACKWARD ? 2 : 1][GN_TPB];
    const int64_t items = p.batch * p.groups;
    const int C = min(p.width, GN_TPB), Q = GN_TPB / C, q = (int)threadIdx.x / C, lane = (int)threadIdx.x % C;      // channels at a time, threads of each
    const double count = (double)p.points * p.width;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t sample = item / p.groups;
        const int c0 = (int)(item - sample * p.groups) * p.width;
        const float *parts = p.part + sample * p.chunks * 2 * p.cols + c0;
        const double k0 = BACKWARD ? 0. : (double)parts[0], rstd = BACKWARD ? p.rstd[item] : 0.f;
        double v[2] = {0., 0.};
        for (int first = 0; first < p.width; first += C) {
            const int c = first + lane;
            const bool on = q < Q && c < p.width;
            double s[2] = {0., 0.};
            if (on) {
                const float *part = parts + c;
#pragma unroll 4
                for (int i = q; i < p.chunks; i += Q) {
                    const float a = part[(int64_t)(2 * i) * p.cols], b = part[(int64_t)(2 * i + 1) * p.cols];
                    if constexpr (BACKWARD) {
                        s[0] += a;
                        s[1] += b;
                    } else {
                        const double n = (double)min(p.rows, p.points - i * p.rows), d = (double)a - k0;
                        s[0] += n * d;
                        s[1] += b + n * d * d;
                    }
                }
            }
            if constexpr (!BACKWARD) {
                v[0] += s[0];
                v[1] += s[1];
            } else {
                __syncthreads();
                col[0][threadIdx.x] = s[0];
                col[1][threadIdx.x] = s[1];
                __syncthreads();
                if (on && q == 0) {
                    for (int i = 1; i < Q; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) s[j] += col[j][i * C + lane];
                    s[1] *= rstd;
                    const double w = p.w ? fe_load(p.w, c0 + c, p.wtype) : 1.f;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        p.sums[(sample * 2 + j) * p.cols + c0 + c] = (float)s[j];
                        v[j] += w * s[j];
                    }
                }
            }
        }
        gn_all<2>(v, red);
        if (threadIdx.x == 0) {
            if constexpr (BACKWARD) {
                p.group[item * 2] = (float)(v[0] / count);
                p.group[item * 2 + 1] = (float)(v[1] / count);
            } else {
                const double mean = v[0] / count, var = v[1] / count - mean * mean;
                p.mean[item] = (float)(k0 + mean);
                p.rstd[item] = (float)(1. / sqrt((var > 0. || var != var ? var : 0.) + (double)p.eps));
            }
        }
    }
}

// y, or dx, of a chunk of points.
template <typename E, bool BACKWARD, int ACT>
__global__ __launch_bounds__(GN_TPB) void gn_apply_kernel(GroupNormP p)
{
    constexpr int V = fe_width<E>, U = 4, WHAT = BACKWARD ? GN_GRADIENT : GN_VALUES;
    typedef typename fe_vec<E>::type vec;
    __shared__ float co[WHAT][GN_TPB * V];
    const uint32_t items = (uint32_t)(p.batch * p.chunks * p.tiles);
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        // the last chunks first: they are the ones that the sums have left in the caches
        const GnPlace o = gn_place<V>(p, items - 1 - item);
        gn_prepare<WHAT, V>(p, o, co);
        if (!o.on) continue;
        const E *x = (const E *)p.x + o.sample * p.sx + o.c;
        const int64_t base = o.sample * p.points * p.cols + o.c;
        float ca[V], cc[V], ce[V], cf[V];
        gn_take<V>(ca, co[0], o);
        gn_take<V>(cc, co[1], o);
        if constexpr (BACKWARD) {
            gn_take<V>(ce, co[2], o);
            gn_take<V>(cf, co[3], o);
        }
        auto finish = [&](vec vx, vec vg, int64_t r) {
            float v[V], z[V];
            gn_floats<E, V>(v, vx);
#pragma unroll
            for (int i = 0; i < V; ++i) z[i] = fmaf(v[i], ca[i], cc[i]);
            if constexpr (BACKWARD) {
                float g[V];
                gn_floats<E, V>(g, vg);
                gm_act_slope(g, z, ACT, p.slope);
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = fmaf(g[i], ca[i], fmaf(v[i], ce[i], cf[i]));
                gm_store<E, V>(g, (E *)p.dx + base + r * p.cols, o.left);
            } else {
                gm_act(z, ACT, p.slope);
                gm_store<E, V>(z, (E *)p.y + base + r * p.cols, o.left);
            }
        };
        int64_t r = o.first + o.row;
        for (; r + (U - 1) * o.step < o.last; r += U * o.step) {
            vec v[U], g[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                v[j] = gn_read<E>(x + (r + j * o.step) * p.ldx, o.left);
                if constexpr (BACKWARD) g[j] = gn_read<E>((const E *)p.gy + base + (r + j * o.step) * p.cols, o.left);
            }
#pragma unroll
            for (int j = 0; j < U; ++j) finish(v[j], g[j], r + j * o.step);
        }
        for (; r < o.last; r += o.step) {
            vec v = gn_read<E>(x + r * p.ldx, o.left), g = {};
            if constexpr (BACKWARD) g = gn_read<E>((const E *)p.gy + base + r * p.cols, o.left);
            finish(v, g, r);
        }
    }
}

// ------------------------------------------------------------------------------------------------ samples that fit a workgroup's registers
// T threads hold the points of a slab (a few whole groups) of one sample, 16 bytes in each of R registers quads a thread, so that everything is read
// once; sums go over the threads through LDS, deviations are taken from the mean itself.  Thread t holds vector t % lanes of points t / lanes + i T / lanes.
struct GroupHeldP { GroupNormP p; int slab, slabs, lanes; int64_t rows; };      // slab: channels; rows: thread groups (places) a slab, and rows of `sums`
template <typename E, int T, int SUMS>
constexpr int gn_held_floats() { return SUMS * (T * fe_width<E> + T) + 2 * T; }        // LDS of T threads

// Sums of v over the points, [threads a channel][the slab's channels] of them to part; K: threads a channel; o: the vector, in the slab.
template <int T, int V>
__device__ __forceinline__ void gn_held_points(const float (&v)[V], float *red, float *part, int t, const GnVector &o, int row, int wide, int steps, int K)
{
    if (row < steps) {
#pragma unroll
        for (int i = 0; i < V; ++i) if (i >= o.shared && i < o.left) red[row * wide + o.c + i] = v[i];
    }
    __syncthreads();
    if (t < K * wide) {
        const int at = t, c = at % wide, k = at / wide;
        float sum = 0.f;
        for (int r = k; r < steps; r += K) sum += red[r * wide + c];
        part[at] = sum;
    }
}
// Sums over the groups' channels (times w where given) to `group`, one wave a group, or one thread where groups are narrow.
template <int T, typename F>
__device__ __forceinline__ void gn_held_groups(const float *part, float *group, int t, int wide, int K, int width, int groups, F f)
{
    if (width * K <= 32) {
        for (int g = t; g < groups; g += T) {
            float sum = 0.f;
            for (int c = 0; c < width; ++c)
                for (int k = 0; k < K; ++k) sum += f(g * width + c) * part[k * wide + g * width + c];
            group[g] = sum;
        }
    } else {
        for (int g = t >> 6; g < groups; g += T / 64) {
            float sum = 0.f;
            for (int i = t & 63; i < width * K; i += 64) sum += f(g * width + i % width) * part[i / width * wide + g * width + i % width];
            sum = fg_wave_sum(sum);
            if ((t & 63) == 0) group[g] = sum;
        }
    }
}

template <typename E, int T, int R, bool BACKWARD>
__global__ __launch_bounds__(T > GN_TPB ? T : GN_TPB) void gn_held_kernel(GroupHeldP h)
{
    typedef typename fe_vec<E>::type vec;
    constexpr int V = fe_width<E>, TPB = T > GN_TPB ? T : GN_TPB, G = TPB / T, SUMS = BACKWARD ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const GroupNormP &p = h.p;
    const int t = (int)threadIdx.x % T, steps = T / h.lanes, r0 = t / h.lanes;
    float *red = lds + (threadIdx.x / T) * gn_held_floats<E, T, SUMS>(), *part = red + SUMS * T * V, *group = part + SUMS * T;
    // neighbouring slabs run on one XCD, whose L2 holds the lines that they share
    const int total = (int)gridDim.x, b = (int)blockIdx.x, xcd = b % FGNN_NUM_XCD, each = total / FGNN_NUM_XCD, rest = total % FGNN_NUM_XCD;
    const int64_t place = ((int64_t)xcd * each + min(xcd, rest) + b / FGNN_NUM_XCD) * G + threadIdx.x / T;
    const int slab = (int)(place % h.slabs), c0 = slab * h.slab, wide = min(p.cols - c0, h.slab), groups = wide / p.width, g0 = c0 / p.width, K = min(steps, T / wide);
    const GnVector own_v = gn_vector<V>(t % h.lanes * V, wide, 0);
    const int c = c0 + own_v.c, left = own_v.left;
    const bool on = r0 < steps && t % h.lanes * V < wide;
    const float inv = 1.f / ((float)p.points * (float)p.width);
    float w[V], bias[V];
    int in[V];                              // the channels' groups, in the slab
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int j = min(c + i, c0 + wide - 1);
        w[i] = p.w ? fe_load(p.w, j, p.wtype) : 1.f;
        bias[i] = p.b ? fe_load(p.b, j, p.btype) : 0.f;
        in[i] = (j - c0) / p.width;
    }
    float own[2] = {0.f, 0.f};              // sums of A and B of the slab's channel t over this place's samples
    const int64_t rounds = (p.batch + h.rows - 1) / h.rows;
    for (int64_t round = 0; round < rounds; ++round) {
        const int64_t sample = place / h.slabs + round * h.rows;
        // (formed again in every round, and before the results: offsets of all points kept over the loop would take the registers of as many points)
        int at = r0;
        asm volatile("" : "+v"(at));
        const bool there = sample < p.batch && place / h.slabs < h.rows;
        const E *x = (const E *)p.x + sample * p.sx + c;
        int64_t base = sample * p.points * p.cols + c;
        const int points = there && on ? (int)p.points : 0;
        vec vx[R], vg[BACKWARD ? R : 1];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            const int r = at + i * steps;
            vx[i] = vec{};
            if constexpr (BACKWARD) vg[i] = vec{};
            if (r < points) {
                vx[i] = gn_read<E>(x + r * p.ldx, left);
                if constexpr (BACKWARD) vg[i] = gn_read<E>((const E *)p.gy + base + (int64_t)r * p.cols, left);
            }
        }
        asm volatile("" : "+v"(base), "+v"(at));
        if constexpr (!BACKWARD) {
            float mean[V], rstd[V];
#pragma unroll
            for (int pass = 0; pass < 2; ++pass) {
                float sum[V];
#pragma unroll
                for (int j = 0; j < V; ++j) sum[j] = 0.f;
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (at + i * steps < points) {
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const float v = (float)vx[i][j] - (pass ? mean[j] : 0.f);
                            sum[j] = pass ? fmaf(v, v, sum[j]) : sum[j] + v;
                        }
                    }
                __syncthreads();            // the sums before are read
                gn_held_points<T, V>(sum, red, part, t, own_v, on ? r0 : steps, wide, steps, K);
                __syncthreads();
                gn_held_groups<T>(part, group, t, wide, K, p.width, groups, [](int) { return 1.f; });
                __syncthreads();
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float v = group[in[j]] * inv;
                    if (pass) rstd[j] = 1.f / sqrtf(v + p.eps);
                    else mean[j] = v;
                }
                if (there)
                    for (int g = t; g < groups; g += T) {
                        const float v = group[g] * inv;
                        if (pass) p.rstd[sample * p.groups + g0 + g] = 1.f / sqrtf(v + p.eps);
                        else p.mean[sample * p.groups + g0 + g] = v;
                    }
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int r = at + i * steps;
                if (r < points) {
                    float v[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) v[j] = fmaf(((float)vx[i][j] - mean[j]) * rstd[j], w[j], bias[j]);
                    gm_act(v, p.act, p.slope);
                    gm_store<E, V>(v, (E *)p.y + base + (int64_t)r * p.cols, left);
                }
            }
        } else {
            GnCols<V> cols;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int64_t g = (there ? sample : 0) * p.groups + g0 + in[j];
                cols.rstd[j] = p.rstd[g];
                cols.mean[j] = -p.mean[g] * cols.rstd[j];
                cols.w[j] = w[j];
                cols.b[j] = bias[j];
            }
            float sum[2][V];
#pragma unroll
            for (int j = 0; j < V; ++j) sum[0][j] = sum[1][j] = 0.f;
            auto terms = [&](int i, float (&u)[V], float (&d)[V]) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    u[j] = (float)vx[i][j];
                    d[j] = (float)vg[i][j];
                }
                gn_slope<V>(p, cols, u, d);
            };
#pragma unroll
            for (int i = 0; i < R; ++i) {
                __builtin_amdgcn_sched_barrier(0);      // one point's terms at a time: the registers are full of points
                if (at + i * steps < points) {
                    float u[V], d[V];
                    terms(i, u, d);
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        sum[0][j] += d[j];
                        sum[1][j] = fmaf(d[j], u[j], sum[1][j]);
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 2; ++k) gn_held_points<T, V>(sum[k], red + k * T * V, part + k * T, t, own_v, on ? r0 : steps, wide, steps, K);
            __syncthreads();
            const auto weight = [&](int j) { return p.w ? fe_load(p.w, c0 + j, p.wtype) : 1.f; };
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                gn_held_groups<T>(part + k * T, group + k * T, t, wide, K, p.width, groups, weight);
                if (t < wide)
                    for (int i = 0; i < K; ++i) own[k] += part[k * T + i * wide + t];
            }
            __syncthreads();
            float ma[V], mb[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ma[j] = group[in[j]] * inv;
                mb[j] = group[T + in[j]] * inv;
            }
            if (p.dx) {
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    const int r = at + i * steps;
                    if (r < points) {
                        float u[V], d[V];
                        terms(i, u, d);
#pragma unroll
                        for (int j = 0; j < V; ++j) d[j] = cols.rstd[j] * (fmaf(d[j], cols.w[j], -ma[j]) - u[j] * mb[j]);
                        gm_store<E, V>(d, (E *)p.dx + base + (int64_t)r * p.cols, left);
                    }
                }
            }
        }
    }
    if (BACKWARD && place / h.slabs < h.rows && t < wide) {
        p.sums[(place / h.slabs * 2) * p.cols + c0 + t] = own[0];
        p.sums[(place / h.slabs * 2 + 1) * p.cols + c0 + t] = own[1];
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
// Whether a sample's slab fits a workgroup: slabs are whole groups, 128 bytes (a cache line) of a point where that fits and more where a wave would hold little, no more
// channels than threads.  T, R: threads and vectors a thread, 0 where nothing fits.
struct GnHeld { GroupHeldP h; int T, R, grid; };
template <typename Fn>
static void gn_held_shape(int T, int R, Fn &&f)
{
    if (T == 64) {
        if (R == 1) f.template operator()<64, 1>();
        else f.template operator()<64, 4>();
    } else if (T == 256) {
        if (R == 2) f.template operator()<256, 2>();
        else if (R == 4) f.template operator()<256, 4>();
        else f.template operator()<256, 8>();
    } else if (R == 8) f.template operator()<512, 8>();
    else if (R == 16) f.template operator()<512, 16>();
    else f.template operator()<512, 18>();
}
static GnHeld gn_held(const GroupNormP &p, int type)
{
    GnHeld o = {};
    const int v = 16 / fe_size(type), width = p.cols / p.groups, cus = fgnn_current_device_compute_units();
    if (width > 512 || p.points > 18 * 512) return o;
    const auto lanes = [&](int groups) { return ((int64_t)groups * width + v - 1) / v; };
    // vectors a thread, for T threads: the points that they hold at a time are whole
    const auto deep = [&](int groups, int T) { return lanes(groups) > T ? (int64_t)1 << 30 : (p.points + T / lanes(groups) - 1) / (T / lanes(groups)); };
    int n = (int)std::min<int64_t>(p.groups, (128 / fe_size(type) + width - 1) / width);
    while (n > 1 && (n * width > 512 || deep(n, 512) > 18)) --n;
    if (deep(n, 512) > 18) return o;
    while (2 * n <= p.groups && 2 * n * width <= 64 && deep(2 * n, 64) <= 1) n *= 2;
    const int64_t d64 = n * width <= 64 ? deep(n, 64) : 1 << 30, d256 = n * width <= 256 ? deep(n, 256) : 1 << 30, d512 = deep(n, 512);
    o.T = d64 <= 4 ? 64 : d256 <= 8 ? 256 : 512;
    o.R = o.T == 64 ? (d64 <= 1 ? 1 : 4) : o.T == 256 ? (d256 <= 2 ? 2 : d256 <= 4 ? 4 : 8) : d512 <= 8 ? 8 : d512 <= 16 ? 16 : 18;
    // 18 vectors a thread: 32 x 1152 x 512 fp32 in 32 groups with silu 33 us forward and 109 in training, 46 and 146 in chunks; 64 x 2176 x 256 bf16 49 and 170 for 58 and 204 (rows of
    // 16 bytes are the other way round, 300 x 9000 x 8 bf16 42 and 160 for 32 and 100).
    // (182 workgroups of 18 vectors a thread, 13 x 1433 x 602 fp16 with gelu: 101 us forward and backward, 90 in chunks)
    if (o.R > 8 && p.batch * ((p.groups + n - 1) / n) < (cus > 0 ? cus : 256)) return GnHeld{};
    o.h.slab = n * width;
    o.h.slabs = (p.groups + n - 1) / n;
    o.h.lanes = (int)lanes(n);
    // every place keeps its slab: as many workgroups as give each slab the same number of places, four times what the device holds at the most
    const int G = std::max(1, GN_TPB / o.T);
    const int64_t wanted = (int64_t)(cus > 0 ? cus : 256) * (o.T == 512 ? 4 : 16) * G;
    o.h.rows = std::max<int64_t>(1, std::min<int64_t>(p.batch, wanted / o.h.slabs));
    o.grid = (int)((o.h.rows * o.h.slabs + G - 1) / G);
    return o;
}
template <bool BACKWARD>
static void gn_held_launch(GnHeld &o, const GroupNormP &p, int type, hipStream_t st)
{
    o.h.p = p;
    o.h.p.width = p.cols / p.groups;
    fe_dispatch(type, [&]<typename E>() {
        gn_held_shape(o.T, o.R, [&]<int T, int R>() {
            constexpr int G = std::max(1, GN_TPB / T), SUMS = BACKWARD ? 2 : 1;
            constexpr size_t bytes = G * gn_held_floats<E, T, SUMS>() * sizeof(float);
            hipLaunchKernelGGL((gn_held_kernel<E, T, R, BACKWARD>), dim3(o.grid), dim3(std::max(T, GN_TPB)), bytes, st, o.h);
        });
    });
}
template <typename Fn>
static void gn_act(int act, Fn &&f)
{
    if (act == GM_RELU) f.template operator()<GM_RELU>();
    else if (act == GM_GELU) f.template operator()<GM_GELU>();
    else if (act == GM_SILU) f.template operator()<GM_SILU>();
    else if (act == GM_LEAKY) f.template operator()<GM_LEAKY>();
    else f.template operator()<GM_NONE>();
}
static unsigned gn_grid(int64_t items) { return (unsigned)std::min<int64_t>(items, GN_GRID); }

static bool gn_limits(int64_t batch, int64_t points, int cols) { return cols <= 1 << 30 && points <= 1LL << 40 && batch <= 1LL << 31; }
static int gn_check(const char *who, int64_t batch, int64_t points, int cols, int groups, int type, const void *x, int64_t ldx, int64_t sx, const void *w, int wtype, const void *b,
                    int btype, int act)
{
    FGNN_REQUIRE(batch >= 0 && points >= 0 && cols >= 1 && groups >= 1 && cols % groups == 0 && ldx >= cols && sx >= 0, FGNN_ERR_SHAPE,
                 "%s: bad sizes batch=%lld points=%lld cols=%d groups=%d ldx=%lld", who, (long long)batch, (long long)points, cols, groups, (long long)ldx);
    FGNN_REQUIRE(fe_is_float(type) && (!w || wtype == type || wtype == FGNN_F32) && (!b || btype == type || btype == FGNN_F32), FGNN_ERR_SHAPE,
                 "%s: element type %d with weights of type %d, bias of type %d", who, type, wtype, btype);
    FGNN_REQUIRE(act >= GM_NONE && act <= GM_LEAKY, FGNN_ERR_SHAPE, "%s: activation %d", who, act);
    FGNN_REQUIRE(gn_limits(batch, points, cols), FGNN_ERR_LIMIT, "%s: batch=%lld points=%lld cols=%d", who, (long long)batch, (long long)points, cols);
    FGNN_REQUIRE(batch == 0 || points == 0 || x, FGNN_ERR_NULL, "%s: NULL argument", who);
    return 0;
}

// The sums of the chunks, then (backward) those of a sample and of a group.
static bool gn_fits(const GroupNormP &p) { return p.batch * p.chunks * p.tiles < 1LL << 31; }
static size_t gn_part_bytes(const GroupNormP &p) { return fgnn_align256((size_t)p.batch * p.chunks * 2 * p.cols * sizeof(float)); }
static size_t gn_sums_bytes(const GroupNormP &p) { return fgnn_align256((size_t)p.batch * 2 * p.cols * sizeof(float)); }
static size_t gn_workspace(int64_t batch, int64_t points, int cols, int groups, int type, int backward)
{
    if (batch < 1 || points < 1 || cols < 1 || groups < 1 || cols % groups || !gn_limits(batch, points, cols) || !fe_is_float(type)) return 0;     // (which a call refuses)
    GroupNormP p = {};
    p.batch = batch; p.points = points; p.cols = cols; p.groups = groups;
    const GnHeld held = gn_held(p, type);
    if (held.T) return backward ? fgnn_align256((size_t)held.h.rows * 2 * cols * sizeof(float)) : 0;
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
    hipStream_t st = (hipStream_t)stream;
    GnHeld held = gn_held(p, type);
    if (held.T) {
        gn_held_launch<false>(held, p, type, st);
        return fgnn_launch_status("gn_held_kernel");
    }
    gn_cut(p, type);
    FGNN_REQUIRE(gn_fits(p), FGNN_ERR_LIMIT, "fgnn_group_norm: %lld samples", (long long)batch);
    FGNN_REQUIRE(workspace && workspace_bytes >= gn_workspace(batch, points, cols, groups, type, 0), FGNN_ERR_WORKSPACE, "fgnn_group_norm: workspace of %zu bytes", workspace_bytes);
    p.part = (float *)workspace;
    const unsigned grid = gn_grid(batch * p.chunks * p.tiles);
    fe_dispatch(type, [&]<typename E>() {
        hipLaunchKernelGGL((gn_moments_kernel<E>), dim3(grid), dim3(GN_TPB), 0, st, p);
        hipLaunchKernelGGL((gn_group_kernel<false>), dim3(gn_grid(batch * groups)), dim3(GN_TPB), 0, st, p);
        gn_act(act, [&]<int ACT>() { hipLaunchKernelGGL((gn_apply_kernel<E, false, ACT>), dim3(grid), dim3(GN_TPB), 0, st, p); });
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
    int64_t rows = empty ? 0 : batch;       // of the sums of dw and db
    GroupNormP p = {batch, points, cols, groups, 0, x, ldx, sx, weight, bias, wtype, btype, 0.f, slope, act, nullptr, const_cast<float *>(mean), const_cast<float *>(rstd), gy, dx};
    if (!weight) p.wtype = type;
    if (!bias) p.btype = type;
    if (!empty) {
        FGNN_REQUIRE(gy && mean && rstd, FGNN_ERR_NULL, "fgnn_group_norm_backward: NULL argument");
        FGNN_REQUIRE(workspace && workspace_bytes >= gn_workspace(batch, points, cols, groups, type, 1), FGNN_ERR_WORKSPACE, "fgnn_group_norm_backward: workspace of %zu bytes",
                     workspace_bytes);
        GnHeld held = gn_held(p, type);
        if (held.T) {
            p.sums = (float *)workspace;
            rows = held.h.rows;
            gn_held_launch<true>(held, p, type, st);
        } else {
            gn_cut(p, type);
            FGNN_REQUIRE(gn_fits(p), FGNN_ERR_LIMIT, "fgnn_group_norm_backward: %lld samples", (long long)batch);
            p.part = (float *)workspace;
            p.sums = (float *)((char *)workspace + gn_part_bytes(p));
            p.group = (float *)((char *)p.sums + gn_sums_bytes(p));
            const unsigned grid = gn_grid(batch * p.chunks * p.tiles);
            fe_dispatch(type, [&]<typename E>() {
                gn_act(act, [&]<int ACT>() { hipLaunchKernelGGL((gn_sums_kernel<E, ACT>), dim3(grid), dim3(GN_TPB), 0, st, p); });
                hipLaunchKernelGGL((gn_group_kernel<true>), dim3(gn_grid(batch * groups)), dim3(GN_TPB), 0, st, p);
                if (dx) gn_act(act, [&]<int ACT>() { hipLaunchKernelGGL((gn_apply_kernel<E, true, ACT>), dim3(grid), dim3(GN_TPB), 0, st, p); });
            });
        }
        const int launched = fgnn_launch_status("gn_apply_kernel");
        if (launched) return launched;
    }
    if (dweight || dbias) {
        hipLaunchKernelGGL(gn_weights_kernel, dim3(gn_grid(2 * (((int64_t)cols + 15) / 16))), dim3(1024), 0, st, p.sums, rows, cols, dweight, p.wtype, dbias, p.btype);
        return fgnn_launch_status("gn_weights_kernel");
    }
    return 0;
}
