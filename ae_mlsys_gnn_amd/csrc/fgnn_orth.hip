// Orthogonalised updates of weight matrices by Newton-Schulz products: X_0 = G / (|G|_F + eps), and each step, with the side s the smaller one,
//     A = X X^T (X^T X for a tall X),   B = b A + c A^2,   X <- a X + B X (X + X B),
// moves every singular value by a s + b s^3 + c s^5.  4 s^2 w + 2 s^3 operations a step for s x w.
//
// A step multiplies rounding errors of small singular values by a (3.4 at the usual coefficients, 490 in five steps), so the products have to carry more than
// 16-bit values do.  X, A and B are kept as two fp16 planes, 22 significant bits, and a product is hi hi + hi lo + lo hi, summed in 32 bits: three
// instructions of the fast kind where fp32 takes sixteen.  The low plane is kept 2^11 times as large: as it is, it would often lie where fp16's step is 2^-24
// whatever the value, with few bits or none (the instructions take subnormal operands as they are).  fp16 has no exponents to spare, so each matrix is scaled
// by a power of two that its largest possible element allows: the singular values of X_0 are at most 1, and what a step makes of the bound is known on the host.
#include <cmath>
#include "fgnn_gemm.h"

typedef _Float16 or_h8 __attribute__((ext_vector_type(8)));

// v = hi + 2^-11 lo, to 2^-23 of v and 2^-36.
__device__ __forceinline__ void or_split(float v, _Float16 &hi, _Float16 &lo)
{
    // v is one value of 32 bits from here on: of a product that was still to be rounded the compiler would form hi twice, for memory from the value of 32 bits and for the
    // difference straight from the product, and one element in 2^13 would get the remainder of another hi
    asm("" : "+v"(v));
    hi = (_Float16)v;
    lo = (_Float16)((v - (float)hi) * 0x1p11f);
}

// One matrix of the iteration in memory: `rows` rows of `cols` columns, padded with zeros to `ld` (whole 16-byte chunks), two planes, a batch of them.
struct OrthM { _Float16 *p; int64_t rows, ld; int cols; };
static __host__ __device__ __forceinline__ int64_t om_plane(const OrthM &m) { return m.rows * m.ld; }

// D = alpha sums + beta C as two planes, or as values of a floating type (`out`, contiguous).
struct OrthEpi {
    static constexpr int W = 8, ROWS = 2;
    OrthM c, d;
    void *out; int type;
    float alpha, beta;
    int mirror;                             // D is symmetric, and what lies further than a tile of so many rows above the diagonal is written from below it; 0: it is not
    struct Cols {};
    __device__ __forceinline__ void columns(int, Cols &) const {}
    struct Ahead { or_h8 hi, lo; };
    __device__ __forceinline__ Ahead ahead(int64_t batch, int64_t m, int n) const
    {
        Ahead a = {};
        if (beta != 0.f) {
            const int64_t plane = d.rows * d.ld, at = batch * 2 * plane + (m < d.rows && n < d.ld ? m * d.ld + n : 0);
            a.hi = *reinterpret_cast<const or_h8 *>(c.p + at);
            a.lo = *reinterpret_cast<const or_h8 *>(c.p + plane + at);
        }
        return a;
    }
    __device__ __forceinline__ void finish(const Cols &, const Ahead &a, int64_t batch, int64_t m, int n, float (&v)[W]) const
    {
        const int64_t plane = d.rows * d.ld;
        if (m >= d.rows || n >= d.ld) return;                   // (rows are whole chunks of eight)
        const int64_t at = batch * 2 * plane + m * d.ld + n;
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] *= alpha;
        if (beta != 0.f) {
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = fmaf(beta, fmaf((float)a.lo[i], 0x1p-11f, (float)a.hi[i]), v[i]);
        }
        const int64_t to = (batch * d.rows + m) * d.cols + n;
        if (out && type == FGNN_F32) gm_store<float, W>(v, (float *)out + to, d.cols - n);
        else if (out && type == FGNN_BF16) gm_store<__bf16, W>(v, (__bf16 *)out + to, d.cols - n);
        else if (out) gm_store<_Float16, W>(v, (_Float16 *)out + to, d.cols - n);
        else {
            or_h8 hi, lo;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                _Float16 a, b;
                or_split(n + i < d.cols ? v[i] : 0.f, a, b);
                hi[i] = a; lo[i] = b;
            }
            *reinterpret_cast<or_h8 *>(d.p + at) = hi;
            *reinterpret_cast<or_h8 *>(d.p + plane + at) = lo;
            if (mirror && n / mirror < m / mirror) {
                // 16 lanes have 16 consecutive m: 32 bytes of a row at a time
#pragma unroll
                for (int i = 0; i < W; ++i)
                    if (n + i < d.cols) {
                        _Float16 *to = d.p + batch * 2 * plane + (n + i) * d.ld + m;
                        to[0] = hi[i];
                        to[plane] = lo[i];
                        if (m == d.rows - 1)                // and the row's padding
                            for (int64_t c = 1; m + c < d.ld; ++c) to[c] = to[plane + c] = (_Float16)0.f;
                    }
            }
        }
    }
};

// The partial sums of a cut reduction, added up in their order: eight columns a thread, 16 rows side by side.
__global__ __launch_bounds__(256) void orth_join_kernel(GemmP p, OrthEpi f)
{
    const int64_t batch = blockIdx.z, m = (int64_t)blockIdx.y * 16 + (threadIdx.x & 15);
    const int n = (int)blockIdx.x * 128 + ((int)threadIdx.x >> 4) * 8;
    if (m >= p.m || n >= p.n || (f.mirror && n / f.mirror > m / f.mirror)) return;
    const OrthEpi::Ahead a = f.ahead(batch, m, n);
    float v[8] = {};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        float u[8];
        gm_load<float, 8>(u, (const float *)p.part + ((batch * p.splits + s) * p.m + m) * p.n + n, p.n - n);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += u[i];
    }
    f.finish({}, a, batch, m, n, v);
}

// ------------------------------------------------------------------------------------------------ norm and planes of X_0
#define OR_PARTS 1024                       // most workgroups that share a matrix's norm
template <typename E>
__global__ __launch_bounds__(256) void orth_norm_kernel(const E *g, int64_t size, float *part)
{
    constexpr int V = fe_width<E>;
    __shared__ float red[4];
    g += (int64_t)blockIdx.y * size;
    float ss = 0.f;
#pragma unroll 4
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < size; i += (int64_t)gridDim.x * 256 * V) {
        float v[V];
        gm_load<E, V>(v, g + i, (int)min((int64_t)V, size - i));
#pragma unroll
        for (int k = 0; k < V; ++k) ss = fmaf(v[k], v[k], ss);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    if (fg_lane() == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    if (threadIdx.x == 0) part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename E>
__global__ __launch_bounds__(256) void orth_planes_kernel(const E *g, const float *part, int parts, float eps, float scale, OrthM x)
{
    __shared__ float red[4];
    float ss = 0.f;
    for (int i = threadIdx.x; i < parts; i += 256) ss += part[(int64_t)blockIdx.y * parts + i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
    if (fg_lane() == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    const float k = scale / (sqrtf((red[0] + red[1]) + (red[2] + red[3])) + eps);
    const int64_t plane = x.rows * x.ld, chunks = plane / 8;
    const int per = (int)(x.ld / 8);
    g += (int64_t)blockIdx.y * x.rows * x.cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per;
        const int col = (int)(i - row * per) * 8;
        float v[8];
        gm_load<E, 8>(v, g + row * x.cols + col, x.cols - col);
        or_h8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            _Float16 a, b;
            or_split(v[j] * k, a, b);
            hi[j] = a; lo[j] = b;
        }
        _Float16 *to = x.p + (int64_t)blockIdx.y * 2 * plane + row * x.ld + col;
        *reinterpret_cast<or_h8 *>(to) = hi;
        *reinterpret_cast<or_h8 *>(to + plane) = lo;
    }
}

static __host__ __device__ __forceinline__ GemmP or_operands(const OrthM &q, bool qs, const OrthM &p, bool ps, int64_t m, int n, int64_t k)
{
    GemmP g{};
    g.m = m; g.n = n; g.k = k;
    g.q = q.p; g.ldq = q.ld; g.rows_q = qs ? (m + 7) / 8 * 8 : m; g.plane_q = om_plane(q) * 2; g.batch_q = 2 * g.plane_q;
    g.p = p.p; g.ldp = p.ld; g.rows_p = ps ? (n + 7) / 8 * 8 : n; g.plane_p = om_plane(p) * 2; g.batch_p = 2 * g.plane_p;
    return g;
}

// ------------------------------------------------------------------------------------------------ small matrices
// All steps of a matrix with a side of at most 128 in one launch: a workgroup goes through the three products of a step, tile by tile, and meets itself in between;
// what it wrote comes back through its own caches.  Bound by the latency of that way, 7 us a tile.
#define OR_STEPS 16
struct OrthFactors { float a, b, b_c, x, x_c; };             // of the epilogues of A, B and X: of the sums, and of what is added
struct OrthSmall {
    OrthM x, y, a, b;
    void *out; int type, steps;
    OrthFactors k[OR_STEPS];
};
// Step i's, chosen among the arguments value by value: a copy of the table would live in memory.
template <int J = 0>
__device__ __forceinline__ void or_factors(const OrthSmall &s, int i, float &a, float &b, float &b_c, float &x, float &x_c)
{
    if constexpr (J < OR_STEPS) {
        const float va = s.k[J].a, vb = s.k[J].b, vbc = s.k[J].b_c, vx = s.k[J].x, vxc = s.k[J].x_c;
        a = i == J ? va : a;
        b = i == J ? vb : b;
        b_c = i == J ? vbc : b_c;
        x = i == J ? vx : x;
        x_c = i == J ? vxc : x_c;
        or_factors<J + 1>(s, i, a, b, b_c, x, x_c);
    }
}
template <bool TALL>
__global__ __launch_bounds__(64 * GM_PLANES_WAVES, 2) void orth_small_kernel(OrthSmall s)
{
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int64_t batch = blockIdx.x;
    const int small = s.a.cols, tiles = (int)(((TALL ? s.x.rows : s.x.cols) + 127) / 128);
#pragma unroll 1
    for (int i = 0; i < s.steps; ++i) {
        OrthM x = s.x, y = s.x;
        x.p = i & 1 ? s.y.p : s.x.p;
        y.p = i & 1 ? s.x.p : s.y.p;
        OrthFactors k{};
        or_factors(s, i, k.a, k.b, k.b_c, k.x, k.x_c);
        GemmP p = TALL ? or_operands(x, true, x, true, small, small, x.rows) : or_operands(x, false, x, false, small, small, x.ld);
        p.splits = 1;
        p.slabs = (p.k + 63) / 64;
        gm_planes_tile<OrthEpi, TALL, TALL>(p, OrthEpi{{}, s.a, nullptr, 0, k.a, 0.f, 0}, 0, 0, 0, batch, lds);
        __syncthreads();
        p = or_operands(s.a, false, s.a, false, small, small, s.a.ld);
        p.splits = 1;
        p.slabs = (p.k + 63) / 64;
        gm_planes_tile<OrthEpi, false, false>(p, OrthEpi{s.a, s.b, nullptr, 0, k.b, k.b_c, 0}, 0, 0, 0, batch, lds);
        __syncthreads();
        const OrthEpi f{x, y, i == s.steps - 1 ? s.out : nullptr, s.type, k.x, k.x_c, 0};
        p = TALL ? or_operands(x, false, s.b, false, x.rows, small, s.b.ld) : or_operands(s.b, false, x, true, small, x.cols, small);
        p.splits = 1;
        p.slabs = (p.k + 63) / 64;
#pragma unroll 1
        for (int t = 0; t < tiles; ++t) {
            gm_planes_tile<OrthEpi, false, !TALL>(p, f, TALL ? t : 0, TALL ? 0 : t, 0, batch, lds);
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------------------------------------ host
// The largest |a s + b s^3 + c s^5| over 0 <= s <= top.
static double or_reach(double a, double b, double c, double top)
{
    auto f = [&](double s) { return std::fabs(s * (a + s * s * (b + s * s * c))); };
    double most = f(top);
    // where the derivative a + 3 b t + 5 c t^2 vanishes, t = s^2
    const double disc = 9 * b * b - 20 * a * c;
    if (c != 0 && disc >= 0) {
        for (int sign = -1; sign <= 1; sign += 2) {
            const double t = (-3 * b + sign * std::sqrt(disc)) / (10 * c);
            if (t > 0 && t < top * top) most = std::max(most, f(std::sqrt(t)));
        }
    } else if (c == 0 && b != 0 && -a / (3 * b) > 0 && -a / (3 * b) < top * top) most = std::max(most, f(std::sqrt(-a / (3 * b))));
    return most;
}
// The largest |b t + c t^2| over 0 <= t <= top.
static double or_reach_b(double b, double c, double top)
{
    double most = std::fabs(top * (b + c * top));
    const double t = c != 0 ? -b / (2 * c) : -1;
    if (t > 0 && t < top) most = std::max(most, std::fabs(t * (b + c * t)));
    return most;
}
// The power of two that leaves elements of at most `bound` a factor of two below fp16's largest value.
static float or_scale(double bound) { return bound > 0 ? (float)std::exp2(std::floor(std::log2(32752.0 / bound))) : 1.f; }

struct OrthShape { int64_t small, wide, ld_x, ld_s; bool tall; int parts; };
static OrthShape or_shape(int64_t m, int64_t n)
{
    OrthShape s{std::min(m, n), std::max(m, n), (n + 7) / 8 * 8, (std::min(m, n) + 7) / 8 * 8, m > n, 0};
    s.parts = (int)std::min<int64_t>(OR_PARTS, (m * n + 8191) / 8192);
    return s;
}

// How a product of D [m, n] over k is laid out: tiles of 256 x 256 where they fill the device or the reduction is long enough to be cut for it, of 128 x 128 else.
struct OrthPlan { int tile, splits; int64_t slabs; };
static OrthPlan or_plan(int64_t m, int64_t n, int64_t k, int batch, bool lower)
{
    const int cus = fgnn_current_device_compute_units(), units = cus > 0 ? cus : 256;
    auto tiles = [&](int64_t t) { const int64_t a = (m + t - 1) / t, b = (n + t - 1) / t; return batch * (lower ? a * (a + 1) / 2 : a * b); };
    const int64_t slabs = (k + 63) / 64;
    auto cut = [&](int64_t t) {
        // (a slab of the reduction is three of the kernel's)
        const int64_t splits = std::max<int64_t>(1, std::min<int64_t>({units / tiles(t), slabs / 4, 16})), each = (slabs + splits - 1) / splits;
        return OrthPlan{(int)t, (int)((slabs + each - 1) / each), each};
    };
    if (tiles(256) >= units) return OrthPlan{256, 1, slabs};
    const OrthPlan big = cut(256);
    return tiles(256) * big.splits * 4 >= units * 3 ? big : cut(128);
}

template <bool QS, bool PS>
static void or_product(GemmP p, OrthEpi f, int batch, bool lower, float *part, hipStream_t st)
{
    const OrthPlan plan = or_plan(p.m, p.n, p.k, batch, lower);
    p.splits = plan.splits; p.slabs = plan.slabs; p.part = part; p.lower = lower;
    f.mirror = lower ? plan.tile : 0;
    p.tiles_m = (int)((p.m + plan.tile - 1) / plan.tile);
    p.tiles_n = (p.n + plan.tile - 1) / plan.tile;
    const int64_t tiles = lower ? (int64_t)p.tiles_m * (p.tiles_m + 1) / 2 : (int64_t)p.tiles_m * p.tiles_n;
    const dim3 grid((unsigned)(tiles * p.splits), (unsigned)batch);
    if (plan.tile == 256)
        hipLaunchKernelGGL((gemm_moved_kernel<FGNN_F16, OrthEpi, QS, PS, 256, 256, 2>), grid, dim3(64 * gm_waves(256, 256)), gm_moved_lds(256, 256), st, p, f);
    else hipLaunchKernelGGL((gemm_planes_kernel<OrthEpi, QS, PS>), grid, dim3(64 * GM_PLANES_WAVES), GM_PLANES_LDS, st, p, f);
    if (p.splits > 1) hipLaunchKernelGGL(orth_join_kernel, dim3((unsigned)((p.n + 127) / 128), (unsigned)((p.m + 15) / 16), (unsigned)batch), dim3(256), 0, st, p, f);
}

// Partial sums of the product that needs the most of them.
static size_t or_part_bytes(int batch, const OrthShape &s, int m, int n)
{
    size_t most = 0;
    auto see = [&](int64_t rows, int64_t cols, int64_t k, bool lower) {
        const OrthPlan p = or_plan(rows, cols, k, batch, lower);
        if (p.splits > 1) most = std::max(most, (size_t)batch * p.splits * rows * cols * sizeof(float));
    };
    see(s.small, s.small, s.tall ? m : s.ld_x, true);
    see(s.small, s.small, s.ld_s, true);
    see(m, n, s.tall ? s.ld_s : s.small, false);
    return most;
}

extern "C" size_t fgnn_orthogonalize_workspace_bytes(int batch, int m, int n)
{
    if (batch < 1 || m < 1 || n < 1) return 0;
    const OrthShape s = or_shape(m, n);
    return (size_t)batch * ((size_t)s.parts * sizeof(float) + 2 * 2 * sizeof(_Float16) * ((size_t)m * s.ld_x + (size_t)s.small * s.ld_s)) + or_part_bytes(batch, s, m, n) + 7 * 256;
}

extern "C" int fgnn_orthogonalize(int batch, int m, int n, int type, const void *g, int steps, const float *coefficients, float eps, void *out, void *workspace,
                                  size_t workspace_bytes, void *stream)
{
    FGNN_REQUIRE(batch >= 0 && m >= 0 && n >= 0 && steps >= 1 && fe_is_float(type), FGNN_ERR_SHAPE, "fgnn_orthogonalize: bad sizes batch=%d m=%d n=%d steps=%d type=%d", batch, m, n,
                 steps, type);
    FGNN_REQUIRE(batch <= 65535 && std::max(m, n) <= (1 << 21), FGNN_ERR_LIMIT, "fgnn_orthogonalize: more than 65535 matrices, or a side of more than 2 M (%d, %d x %d)", batch, m, n);
    if (batch == 0 || m == 0 || n == 0) return 0;
    FGNN_REQUIRE(g && out && coefficients, FGNN_ERR_NULL, "fgnn_orthogonalize: NULL argument");
    FGNN_REQUIRE(workspace && workspace_bytes >= fgnn_orthogonalize_workspace_bytes(batch, m, n), FGNN_ERR_WORKSPACE, "fgnn_orthogonalize: workspace of %zu bytes", workspace_bytes);
    double reach = 1.001;
    for (int i = 0; i < steps; ++i) {
        const float *c = coefficients + 3 * i;
        reach = or_reach(c[0], c[1], c[2], reach) * 1.001;
        FGNN_REQUIRE(reach < 100.0, FGNN_ERR_LIMIT, "fgnn_orthogonalize: the coefficients take a singular value to %g in step %d", reach, i + 1);
    }
    const OrthShape s = or_shape(m, n);
    hipStream_t st = (hipStream_t)stream;
    char *at = (char *)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
    auto take = [&](size_t bytes) { char *p = at; at += fgnn_align256(bytes); return p; };
    auto matrix = [&](int64_t rows, int cols, int64_t ld) { return OrthM{(_Float16 *)take((size_t)batch * 2 * rows * ld * sizeof(_Float16)), rows, ld, cols}; };
    OrthM x = matrix(m, n, s.ld_x), y = matrix(m, n, s.ld_x), a = matrix(s.small, (int)s.small, s.ld_s), b = matrix(s.small, (int)s.small, s.ld_s);
    float *norms = (float *)take((size_t)batch * s.parts * sizeof(float)), *part = (float *)take(or_part_bytes(batch, s, m, n));

    double top = 1.001;
    float sx = or_scale(top);
    fe_dispatch(type, [&]<typename E>() {
        hipLaunchKernelGGL((orth_norm_kernel<E>), dim3(s.parts, batch), dim3(256), 0, st, (const E *)g, (int64_t)m * n, norms);
        const unsigned blocks = (unsigned)std::min<int64_t>((om_plane(x) / 8 + 255) / 256, 4096);
        hipLaunchKernelGGL((orth_planes_kernel<E>), dim3(blocks, batch), dim3(256), 0, st, (const E *)g, (const float *)norms, s.parts, eps, sx, x);
    });
    // One launch for all steps where a workgroup's way through the tiles of X is no longer than the launches, or there are many matrices (us, launches / one: one of
    // 64 x 64 94 / 65, four of 128 x 256 155 / 154, one of 128 x 512 167 / 248, 100 of them 345 / 276, 300 of 100 x 128 629 / 219).
    const bool one = s.small <= 128 && steps <= OR_STEPS && (s.wide <= 256 || (s.wide <= 512 && batch >= 64));
    OrthSmall all{x, y, a, b, out, type, steps, {}};
    for (int i = 0; i < steps; ++i) {
        const float *c = coefficients + 3 * i;
        const bool last = i == steps - 1;
        const float sa = or_scale(top * top), sb = or_scale(or_reach_b(c[1], c[2], top * top));
        top = or_reach(c[0], c[1], c[2], top) * 1.001;
        const float sy = last ? 1.f : or_scale(top);
        const float alpha[3] = {sa / (sx * sx), sb * c[2] / (sa * sa), sy / (sb * sx)}, beta[3] = {0.f, sb * c[1] / sa, sy * c[0] / sx};
        sx = sy;
        if (one) {
            all.k[i] = OrthFactors{alpha[0], alpha[1], beta[1], alpha[2], beta[2]};
            continue;
        }
        const int small = (int)s.small;
        OrthEpi f{{}, a, nullptr, type, alpha[0], beta[0], 0};
        if (s.tall) or_product<true, true>(or_operands(x, true, x, true, small, small, m), f, batch, true, part, st);
        else or_product<false, false>(or_operands(x, false, x, false, small, small, s.ld_x), f, batch, true, part, st);
        f = OrthEpi{a, b, nullptr, type, alpha[1], beta[1], 0};
        or_product<false, false>(or_operands(a, false, a, false, small, small, s.ld_s), f, batch, true, part, st);
        f = OrthEpi{x, y, last ? out : nullptr, type, alpha[2], beta[2], 0};
        if (s.tall) or_product<false, false>(or_operands(x, false, b, false, m, small, s.ld_s), f, batch, false, part, st);
        else or_product<false, true>(or_operands(b, false, x, true, small, n, small), f, batch, false, part, st);
        std::swap(x, y);
    }
    if (one && s.tall) hipLaunchKernelGGL(orth_small_kernel<true>, dim3(batch), dim3(64 * GM_PLANES_WAVES), GM_PLANES_LDS, st, all);
    else if (one) hipLaunchKernelGGL(orth_small_kernel<false>, dim3(batch), dim3(64 * GM_PLANES_WAVES), GM_PLANES_LDS, st, all);
    return fgnn_launch_status("gemm_moved_kernel");
}
