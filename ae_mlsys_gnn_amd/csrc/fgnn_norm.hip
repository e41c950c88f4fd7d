// Root-mean-square norm of rows with the residual's addition:
//   h = x + r,   s = (mean_j h_j^2 + eps)^-1/2,   y_j = h_j s w_j
// written as values, or in 8 bits with a scale a row (scale = max_j |y_j| / Q, q_j = round(y_j / scale), Q = 127 or 448), and its gradient
//   g = gy w,   dx = dr = gh + s g - h s^3 mean_j(g h),   dw_j = sum_i gy_ij h_ij s_i .
// All three are bound by memory: a row is read once into registers, its statistics (32 bits) are taken from there, and it is written
// once (16,384 x 4096 bf16 with residual, forward and backward 4.8 TB/s; a copy of 1 GiB reaches 5.1).  T threads share a row, R 16-byte vectors each, so that a row of 16 bytes and one of 64 KB keep about as many loads in flight.
#include <algorithm>
#include "fgnn_elem.h"

#define NM_TPB 256
struct NormP {
    int64_t rows;
    int cols, norm;                         // norm 0: y = h (rows are only put into 8 bits)
    const void *x; int64_t ldx;
    const void *r; int64_t ldr;             // residual, or NULL
    const void *w; int wtype;               // weights, or NULL: ones
    float eps, top;                         // top: largest value in 8 bits
    void *h, *y;                            // contiguous; h NULL: not wanted
    float *rstd, *scale;                    // rstd NULL: not wanted
};
struct NormB {
    int64_t rows;
    int cols;
    const void *gy, *gh;                    // contiguous; either may be NULL: zeros
    const void *h; int64_t ldh;
    const void *w; int wtype;
    const float *rstd;
    void *dx;                               // NULL: not wanted
    float *part;                            // [grid][cols], NULL: dw is not wanted
};

// The sum or the maximum over the T threads of a row; every thread gets it.  red: one float a wave and row group.
template <int T, bool MAX>
__device__ __forceinline__ float nm_all(float v, float *red)
{
#pragma unroll
    for (int o = (T < 64 ? T : 64) / 2; o > 0; o >>= 1) {
        const float u = __shfl_xor(v, o, 64);
        v = MAX ? fmaxf(v, u) : v + u;
    }
    if constexpr (T > 64) {
        __syncthreads();                    // the values of the sum before are read
        if (fg_lane() == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < T / 64; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
    }
    return v;
}

template <typename E, int V>
__device__ __forceinline__ void nm_load(float (&v)[V], const E *row, int at, int cols)
{
    if (at + V <= cols) {
        const typename fe_vec<E>::type u = *reinterpret_cast<const typename fe_vec<E>::type *>(row + at);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)u[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = at + i < cols ? (float)row[at + i] : 0.f;
    }
}
template <typename E, int V>
__device__ __forceinline__ void nm_store(const float (&v)[V], E *row, int at, int cols)
{
    if (at + V <= cols) {
        typename fe_vec<E>::type u;
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = (E)v[i];
        *reinterpret_cast<typename fe_vec<E>::type *>(row + at) = u;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (at + i < cols) row[at + i] = (E)v[i];
    }
}
// V values in 8 bits, nearest, ties to even.  Below top * (1 + 2^-22), so that neither form leaves its range.
template <int Q, int V>
__device__ __forceinline__ void nm_store8(const float (&v)[V], uint8_t *row, int at, int cols)
{
    typedef uint32_t words __attribute__((ext_vector_type(V / 4), aligned(1)));
    words u;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        if constexpr (Q == FGNN_I8) {
            uint32_t b = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) b |= ((uint32_t)(int)rintf(v[4 * i + k]) & 255u) << (8 * k);
            u[i] = b;
        } else {
            int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
            u[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], b, true);
        }
    }
    if (at + V <= cols) *reinterpret_cast<words *>(row + at) = u;
    else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (at + i < cols) row[at + i] = (uint8_t)(u[i / 4] >> (8 * (i % 4)));
    }
}

template <typename E, int T, int R, int Q>
__global__ __launch_bounds__(T > NM_TPB ? T : NM_TPB) void norm_kernel(NormP p)
{
    constexpr int V = fe_width<E>, TPB = T > NM_TPB ? T : NM_TPB;
    __shared__ float red[TPB / 64];
    const int lane = (int)threadIdx.x % T;
    const int64_t group = (int64_t)blockIdx.x * (TPB / T) + threadIdx.x / T, groups = (int64_t)gridDim.x * (TPB / T);
    float w[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (r * T + lane) * V + i;
            w[r][i] = p.w && c < p.cols ? fe_load(p.w, c, p.wtype) : 1.f;
        }
    for (int64_t row = group; row < p.rows; row += groups) {
        const E *x = (const E *)p.x + row * p.ldx, *res = (const E *)p.r + row * p.ldr;
        float v[R][V], ss = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * T + lane) * V;
            nm_load<E, V>(v[r], x, c, p.cols);
            if (p.r) {
                float u[V];
                nm_load<E, V>(u, res, c, p.cols);
#pragma unroll
                for (int i = 0; i < V; ++i) v[r][i] += u[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) ss = fmaf(v[r][i], v[r][i], ss);
        }
        if (p.h) {
#pragma unroll
            for (int r = 0; r < R; ++r) nm_store<E, V>(v[r], (E *)p.h + row * p.cols, (r * T + lane) * V, p.cols);
        }
        float s = 1.f;
        if (p.norm) {
            ss = nm_all<T, false>(ss, red);
            s = 1.f / sqrtf(ss / (float)p.cols + p.eps);
            if (p.rstd && lane == 0) p.rstd[row] = s;
        }
        float most = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                v[r][i] = v[r][i] * s * w[r][i];
                // (a NaN is lost in the maximum: the sum of squares has it, and the product with s hands it to every element; without the norm it
                // is looked for)
                if (Q) most = fmaxf(most, v[r][i] == v[r][i] ? fabsf(v[r][i]) : __builtin_inff());
            }
        if constexpr (Q == 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) nm_store<E, V>(v[r], (E *)p.y + row * p.cols, (r * T + lane) * V, p.cols);
        } else {
            most = nm_all<T, true>(most, red);
            // rows of zeros (or of less than 1.4e-36, whose scale has no reciprocal in 32 bits) have scale 0; a row with an infinity or a NaN
            // scale NaN and zeros, so that all of it is NaN to a reader
            const bool finite = most < __builtin_inff(), some = finite && p.top / most < __builtin_inff();
            const float inv = some ? p.top / most : 0.f;
            if (lane == 0) p.scale[row] = some ? most / p.top : finite ? 0.f : __builtin_nanf("");
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int c = (r * T + lane) * V;
                float u[V];
#pragma unroll
                for (int i = 0; i < V; ++i) u[i] = some ? fminf(fmaxf(v[r][i] * inv, -p.top), p.top) : 0.f;
                nm_store8<Q, V>(u, (uint8_t *)p.y + row * p.cols, c, p.cols);
            }
        }
    }
}

// A thread keeps its columns over all rows of its workgroup: their sums of gy h s stay in its registers, and one row of sums a workgroup
// goes to memory, added up by the kernel below in a fixed order.
template <typename E, int T, int R>
__global__ __launch_bounds__(T > NM_TPB ? T : NM_TPB) void norm_backward_kernel(NormB p)
{
    constexpr int V = fe_width<E>, TPB = T > NM_TPB ? T : NM_TPB, G = TPB / T;
    __shared__ float red[TPB / 64], sums[G > 1 ? TPB * V * R : 1];
    const int lane = (int)threadIdx.x % T;
    const int64_t group = (int64_t)blockIdx.x * G + threadIdx.x / T, groups = (int64_t)gridDim.x * G;
    float w[R][V], dw[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (r * T + lane) * V + i;
            w[r][i] = p.w && c < p.cols ? fe_load(p.w, c, p.wtype) : 1.f;
            dw[r][i] = 0.f;
        }
    const float inv = 1.f / (float)p.cols;
    for (int64_t row = group; row < p.rows; row += groups) {
        float g[R][V], h[R][V], dot = 0.f;
        const float s = p.rstd[row];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * T + lane) * V;
            nm_load<E, V>(h[r], (const E *)p.h + row * p.ldh, c, p.cols);
            if (p.gy) nm_load<E, V>(g[r], (const E *)p.gy + row * p.cols, c, p.cols);
            else {
#pragma unroll
                for (int i = 0; i < V; ++i) g[r][i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dw[r][i] = fmaf(g[r][i], h[r][i] * s, dw[r][i]);
                g[r][i] *= w[r][i];
                dot = fmaf(g[r][i], h[r][i], dot);
            }
        }
        if (!p.dx) continue;
        dot = nm_all<T, false>(dot, red);
        const float k = s * s * (s * dot * inv);           // (s dot is of the gradient's size, where s^3 leaves 32 bits for rows of 1e13 or 1e-13)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * T + lane) * V;
            float d[V];
            if (p.gh) nm_load<E, V>(d, (const E *)p.gh + row * p.cols, c, p.cols);
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = s * g[r][i] - h[r][i] * k + (p.gh ? d[i] : 0.f);
            nm_store<E, V>(d, (E *)p.dx + row * p.cols, c, p.cols);
        }
    }
    if (!p.part) return;
    if constexpr (G > 1) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < V; ++i) sums[(threadIdx.x / T) * (T * V * R) + (r * T + lane) * V + i] = dw[r][i];
        __syncthreads();
        for (int c = threadIdx.x; c < p.cols; c += TPB) {
            float v = 0.f;
#pragma unroll 4
            for (int i = 0; i < G; ++i) v += sums[i * (T * V * R) + c];
            p.part[(int64_t)blockIdx.x * p.cols + c] = v;
        }
    } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = (r * T + lane) * V + i;
                if (c < p.cols) p.part[(int64_t)blockIdx.x * p.cols + c] = dw[r][i];
            }
    }
}

// out [cols] = the column sums of part [rows, cols], in a type known at run time: 16 columns a workgroup at a time, 64 rows side by side.  Summed in 64 bits and rounded
// once: as many as 1024 parts, 64 of their sums one after the other, in 32 bits were off by more than all sums before them, and no faster (1024 parts of 4096
// columns 7.3 us, in 64 bits 7.1; 170 of 128 3.4 / 3.4).
#define NM_SUM_GRID (1 << 20)               // most workgroups: a launch has fewer than 2^32 threads
__global__ __launch_bounds__(1024) void norm_sum_kernel(const float *__restrict__ part, int rows, int cols, void *out, int type)
{
    __shared__ double red[16][17];
    const int c = (int)threadIdx.x & 15, q = (int)threadIdx.x >> 4;
    for (int64_t first = (int64_t)blockIdx.x * 16; first < cols; first += (int64_t)gridDim.x * 16) {
        const int64_t col = first + c;
        double v = 0.;
        if (col < cols) {
#pragma unroll 4
            for (int i = q; i < rows; i += 64) v += part[(int64_t)i * cols + col];
        }
        // the four sums of a wave, then those of the 16 waves
        v += __shfl_xor(v, 16, 64);
        v += __shfl_xor(v, 32, 64);
        __syncthreads();                    // the sums before are read
        if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][c] = v;
        __syncthreads();
        if (threadIdx.x < 64) {
            v = 0.;
#pragma unroll
            for (int i = 0; i < 4; ++i) v += red[4 * i + q][c];
            v += __shfl_xor(v, 16, 64);
            v += __shfl_xor(v, 32, 64);
            if (q == 0 && col < cols) fe_store(out, col, type, (float)v);
        }
    }
}

int fgnn_sum_parts(const float *part, int rows, int cols, void *out, int type, hipStream_t st)
{
    const unsigned groups = (unsigned)(((int64_t)cols + 15) / 16);
    hipLaunchKernelGGL(norm_sum_kernel, dim3(std::min<unsigned>(groups, NM_SUM_GRID)), dim3(1024), 0, st, part, rows, cols, out, type);
    return fgnn_launch_status("norm_sum_kernel");
}

// Threads a row and vectors a thread; columns that are no multiple of the vector take part of one.  Rows of 65 to 96 vectors that become 8 bits take half a
// wave: their two reductions and short stores cost more than idle lanes in the loads (100,000 rows of fp16, us, 64 threads / 32: 520 columns 117 / 105, 602 157 / 130, 768
// 142 / 121; as values 86 / 114, 112 / 145, 117 / 141; backward 130 / 176, 187 / 228, 148 / 190).  Above 512 vectors registers decide, the backward pass's
// most (14,000 rows of fp16, us, 256 threads / as below: 4736 columns as values 131 / 104, 8 bits 143 / 126, backward 232 / 198; 8192 187 / 171, 174 / 174, 295 / 217; with
// 1024 threads of four vectors / of two: 12,000 374 / 283, 533 / 324, 1815 / 348).
enum { NM_FORWARD, NM_EIGHT, NM_BACKWARD };
template <int PASS, typename Fn>
static bool nm_shape(int64_t vectors, Fn &&f)
{
    if (vectors <= 16) f.template operator()<16, 1>();
    else if (vectors <= 32) f.template operator()<16, 2>();
    else if (vectors <= 64) f.template operator()<64, 1>();
    else if (vectors <= 128) {
        if constexpr (PASS == NM_EIGHT) {
            if (vectors <= 96) f.template operator()<32, 3>();
            else f.template operator()<64, 2>();
        } else f.template operator()<64, 2>();
    } else if (vectors <= 256) f.template operator()<256, 1>();
    else if (vectors <= 512) f.template operator()<256, 2>();
    else if (vectors <= 1024) {
        if constexpr (PASS == NM_FORWARD) f.template operator()<512, 2>();
        else if constexpr (PASS == NM_BACKWARD) f.template operator()<1024, 1>();
        else if (vectors <= 768) f.template operator()<256, 3>();
        else f.template operator()<256, 4>();
    } else if (vectors <= 2048) f.template operator()<1024, 2>();
    else if (vectors <= 4096) f.template operator()<1024, 4>();
    else return false;
    return true;
}
static inline int nm_vectors(int cols, int type) { const int v = 16 / fe_size(type); return (cols + v - 1) / v; }
// per_unit: workgroups of 256 threads a compute unit
static unsigned nm_grid(int64_t rows, int T, int per_unit)
{
    const int cus = fgnn_current_device_compute_units(), groups = T >= NM_TPB ? 1 : NM_TPB / T;
    return (unsigned)std::min<int64_t>((rows + groups - 1) / groups, (int64_t)(cus > 0 ? cus : 256) * std::max(1, per_unit * NM_TPB / std::max(T, NM_TPB)));
}

static int nm_check(const char *who, int64_t rows, int cols, int type, const void *x, int64_t ldx, const void *r, int64_t ldr, const void *w, int wtype)
{
    FGNN_REQUIRE(rows >= 0 && cols >= 1 && ldx >= cols && (!r || ldr >= cols), FGNN_ERR_SHAPE, "%s: bad sizes rows=%lld cols=%d ldx=%lld ldr=%lld", who,
                 (long long)rows, cols, (long long)ldx, (long long)ldr);
    FGNN_REQUIRE(fe_is_float(type) && (!w || wtype == type || wtype == FGNN_F32), FGNN_ERR_SHAPE, "%s: element type %d with weights of type %d", who, type, wtype);
    FGNN_REQUIRE(nm_vectors(cols, type) <= 4096, FGNN_ERR_LIMIT, "%s: rows of more than 64 KB (%d columns)", who, cols);
    FGNN_REQUIRE(rows == 0 || x, FGNN_ERR_NULL, "%s: NULL argument", who);
    return 0;
}

static int nm_forward(const char *who, NormP p, int type, int eight, hipStream_t st)
{
    if (p.rows == 0) return 0;
    const int vectors = nm_vectors(p.cols, type);
    fe_dispatch(type, [&]<typename E>() {
        auto launch = [&]<int Q, int T, int R>() {
            hipLaunchKernelGGL((norm_kernel<E, T, R, Q>), dim3(nm_grid(p.rows, T, 8)), dim3(T > NM_TPB ? T : NM_TPB), 0, st, p);
        };
        if (eight == FGNN_I8) nm_shape<NM_EIGHT>(vectors, [&]<int T, int R>() { launch.template operator()<FGNN_I8, T, R>(); });
        else if (eight == FGNN_E4M3) nm_shape<NM_EIGHT>(vectors, [&]<int T, int R>() { launch.template operator()<FGNN_E4M3, T, R>(); });
        else nm_shape<NM_FORWARD>(vectors, [&]<int T, int R>() { launch.template operator()<0, T, R>(); });
    });
    return fgnn_launch_status(who);
}

extern "C" int fgnn_rms_norm(int64_t rows, int cols, int type, const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *weight, int wtype,
                             float eps, void *h, void *y, float *rstd, void *stream)
{
    const int rc = nm_check("fgnn_rms_norm", rows, cols, type, x, ldx, residual, ldr, weight, wtype);
    if (rc) return rc;
    FGNN_REQUIRE(rows == 0 || (y && (!residual || h)), FGNN_ERR_NULL, "fgnn_rms_norm: NULL argument");
    NormP p{rows, cols, 1, x, ldx, residual, ldr, weight, wtype, eps, 0.f, residual ? h : nullptr, y, rstd, nullptr};
    return nm_forward("norm_kernel", p, type, 0, (hipStream_t)stream);
}

extern "C" int fgnn_rms_norm_q8(int64_t rows, int cols, int type, const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *weight, int wtype,
                                float eps, int eight, void *h, void *q, float *scale, void *stream)
{
    const int rc = nm_check("fgnn_rms_norm_q8", rows, cols, type, x, ldx, residual, ldr, weight, wtype);
    if (rc) return rc;
    FGNN_REQUIRE(fe_is_eight(eight), FGNN_ERR_SHAPE, "fgnn_rms_norm_q8: output type %d", eight);
    FGNN_REQUIRE(rows == 0 || (q && scale && (!residual || h)), FGNN_ERR_NULL, "fgnn_rms_norm_q8: NULL argument");
    NormP p{rows, cols, 1, x, ldx, residual, ldr, weight, wtype, eps, fe_top(eight), residual ? h : nullptr, q, nullptr, scale};
    return nm_forward("norm_kernel", p, type, eight, (hipStream_t)stream);
}

extern "C" int fgnn_quantize_rows(int64_t rows, int cols, int type, const void *x, int64_t ldx, int eight, void *q, float *scale, void *stream)
{
    const int rc = nm_check("fgnn_quantize_rows", rows, cols, type, x, ldx, nullptr, 0, nullptr, type);
    if (rc) return rc;
    FGNN_REQUIRE(fe_is_eight(eight), FGNN_ERR_SHAPE, "fgnn_quantize_rows: output type %d", eight);
    FGNN_REQUIRE(rows == 0 || (q && scale), FGNN_ERR_NULL, "fgnn_quantize_rows: NULL argument");
    NormP p{rows, cols, 0, x, ldx, nullptr, 0, nullptr, type, 0.f, fe_top(eight), nullptr, q, nullptr, scale};
    return nm_forward("norm_kernel", p, type, eight, (hipStream_t)stream);
}

static unsigned nm_backward_grid(int64_t rows, int cols, int type)
{
    unsigned grid = 1;
    nm_shape<NM_BACKWARD>(nm_vectors(cols, type), [&]<int T, int R>() { grid = nm_grid(rows, T, 4); });
    return grid;
}

extern "C" size_t fgnn_rms_norm_backward_workspace_bytes(int64_t rows, int cols, int type)
{
    if (rows < 1 || cols < 1 || !fe_is_float(type) || nm_vectors(cols, type) > 4096) return 0;
    return (size_t)nm_backward_grid(rows, cols, type) * cols * sizeof(float);
}

extern "C" int fgnn_rms_norm_backward(int64_t rows, int cols, int type, const void *gy, const void *gh, const void *h, int64_t ldh, const void *weight, int wtype,
                                      const float *rstd, void *dx, void *dweight, void *workspace, size_t workspace_bytes, void *stream)
{
    const int rc = nm_check("fgnn_rms_norm_backward", rows, cols, type, h, ldh, nullptr, 0, weight, wtype);
    if (rc) return rc;
    FGNN_REQUIRE(rows == 0 || rstd, FGNN_ERR_NULL, "fgnn_rms_norm_backward: NULL argument");
    FGNN_REQUIRE(!dweight || rows == 0 || (workspace && workspace_bytes >= fgnn_rms_norm_backward_workspace_bytes(rows, cols, type)), FGNN_ERR_WORKSPACE,
                 "fgnn_rms_norm_backward: workspace of %zu bytes", workspace_bytes);
    hipStream_t st = (hipStream_t)stream;
    int parts = 0;
    if (rows > 0 && (dx || dweight)) {
        NormB p{rows, cols, gy, gh, h, ldh, weight, wtype, rstd, dx, dweight ? (float *)workspace : nullptr};
        parts = (int)nm_backward_grid(rows, cols, type);
        fe_dispatch(type, [&]<typename E>() {
            nm_shape<NM_BACKWARD>(nm_vectors(cols, type), [&]<int T, int R>() {
                hipLaunchKernelGGL((norm_backward_kernel<E, T, R>), dim3(parts), dim3(T > NM_TPB ? T : NM_TPB), 0, st, p);
            });
        });
        const int launched = fgnn_launch_status("norm_backward_kernel");
        if (launched) return launched;
    }
    return dweight ? fgnn_sum_parts((const float *)workspace, parts, cols, dweight, weight ? wtype : type, st) : 0;
}
