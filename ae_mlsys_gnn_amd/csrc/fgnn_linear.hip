// Linear maps with bias, activation and residual in the product's epilogue, and what their gradient needs:
//     z = x W^T + b,  y = act(z) + r;      dz = gy act'(z),  db = sum_i dz_i,  dx = dz W,  dW = dz^T x .
// The products are those of fgnn_gemm.h.  z is kept for the backward pass in the rows' type: the slope of an activation changes by less than z itself does
// by that rounding.
#include "fgnn_gemm.h"

// Columns of a result are counted in 32 bits, up to the end of the tile or strip (of 2048) that holds the last.
#define GM_MOST_COLUMNS (INT32_MAX - 4095)
// A launch has fewer than 2^32 threads.
static bool gm_launches(int64_t workgroups, int threads) { return workgroups < (1ll << 32) / threads; }
static int gm_units() { const int cus = fgnn_current_device_compute_units(); return cus > 0 ? cus : 256; }
static int gm_slab_of(int kind) { return kind == FGNN_F32 ? 32 : kind == FGNN_I8 ? 128 : 64; }

// How a reduction is cut so that a small result still fills the device, four slabs a part at the least.  The kernel that moves its operands to LDS by itself
// fills a compute unit with one workgroup (2048^3 bf16 26.7 us, cut in two for two workgroups 39.5), the one that converts them wants two (fp32 118 / 97).
static void gm_cut(GemmP *p, int tile, int kind, bool moved)
{
    p->tiles_m = (int)((p->m + tile - 1) / tile);
    p->tiles_n = (p->n + tile - 1) / tile;
    const int slab = gm_slab_of(kind), fill = (moved ? 1 : 2) * gm_units();
    const int64_t tiles = (int64_t)p->tiles_m * p->tiles_n, slabs = (p->k + slab - 1) / slab;
    int64_t splits = 1;
    if (tiles > 0 && tiles < fill) splits = std::max<int64_t>(1, std::min<int64_t>({fill / tiles, slabs / 4, 256}));
    p->slabs = std::max<int64_t>(1, (slabs + splits - 1) / splits);
    p->splits = (int)std::max<int64_t>(1, (slabs + p->slabs - 1) / p->slabs);
}

// ------------------------------------------------------------------------------------------------ operands laid out anew
// Rows of 16-bit values, or of 8-bit floats as fp16, copied to rows of whole 16-byte chunks with zeros behind: a chunk a thread.
template <bool E4M3>
__global__ __launch_bounds__(256) void linear_pack_kernel(const char *from, int64_t ld, int64_t rows, int cols, char *to)
{
    const int chunks = (cols + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / chunks;
    if (row >= rows) return;
    const int c = (int)(i - row * chunks) * 8, count = cols - c;
    gm_i4 v = {0, 0, 0, 0};
    if constexpr (E4M3) {
        const uint8_t *p = (const uint8_t *)from + row * ld + c;
        uint32_t w[4] = {0, 0, 0, 0};
        if (count >= 8) __builtin_memcpy(w, p, 8);
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k < count) w[k / 4] |= (uint32_t)p[k] << (8 * (k % 4));
        }
        gm_i4 half[2];
        gm_widen(w, half);
        v = half[0];
    } else {
        const uint16_t *p = (const uint16_t *)from + row * ld + c;
        if (count >= 8) __builtin_memcpy(&v, p, 16);
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k < count) v[k / 2] |= (int)p[k] << (16 * (k % 2));
        }
    }
    reinterpret_cast<gm_i4 *>(to)[i] = v;
}
static size_t gm_packed_bytes(int64_t rows, int64_t cols) { return fgnn_align256((size_t)rows * ((cols + 7) / 8) * 16); }
static int64_t gm_pack_workgroups(int64_t rows, int64_t cols) { return (rows * ((cols + 7) / 8) + 255) / 256; }
static void gm_pack(const void *from, int64_t ld, int64_t rows, int cols, char *to, bool e4m3, hipStream_t st)
{
    const dim3 g((unsigned)gm_pack_workgroups(rows, cols));
    if (e4m3) hipLaunchKernelGGL(linear_pack_kernel<true>, g, dim3(256), 0, st, (const char *)from, ld, rows, cols, to);
    else hipLaunchKernelGGL(linear_pack_kernel<false>, g, dim3(256), 0, st, (const char *)from, ld, rows, cols, to);
}
// Whether a product is large enough for operands that cannot be moved as they lie to be laid out anew first.  us, through registers / laid out and moved,
// forward, input and weights' gradient: 1003^3 (1e9 products) 21 / 27, 24 / 28, 27 / 27; 2049 x 513 -> 2049 (2e9) 27 / 29, 33 / 30, 34 / 30; 5003 x 602 -> 1433
// (4e9) 30 / 29, 54 / 35, 51 / 37; 169,343 x 129 -> 257 (6e9) 101 / 108, 94 / 89, 150 / 101; 8191 x 4097 -> 4095 399 / 270, 546 / 325, 1106 / 408; 8-bit
// floats 8192 x 4096 -> 8192 577 / 407.
static bool gm_worth_packing(int64_t m, int64_t n, int64_t k, int kind)
{
    return (kind == FGNN_BF16 || kind == FGNN_F16 || kind == FGNN_E4M3) && (double)m * n * k >= 3e9;
}

// Whether rows `ld` bytes apart are near enough for the 32-bit offsets of the kernel that moves them: a tile takes up to 256 rows of an operand whose reduction
// is contiguous, 64 of a strided one.
static bool gm_near(int64_t ld, bool strided) { return ld * (strided ? 64 : 256) < (1ll << 31); }
// Whether operands that cannot be moved as they lie are laid out anew: where it is worth it, their new rows are near enough, and a launch has the threads.
static bool gm_packs(int64_t m, int64_t n, int64_t k, int kind, bool qs, bool ps)
{
    return gm_worth_packing(m, n, k, kind) && gm_near(((qs ? m : k) + 7) / 8 * 16, qs) && gm_near(((ps ? n : k) + 7) / 8 * 16, ps)
        && gm_launches(qs ? gm_pack_workgroups(k, m) : gm_pack_workgroups(m, k), 256) && gm_launches(ps ? gm_pack_workgroups(k, n) : gm_pack_workgroups(n, k), 256);
}

// Whether rows of an operand are whole 16-byte chunks at 16-byte addresses, and near enough.
// (padded: zeros follow a row up to whole chunks)
static bool gm_movable(const void *p, int64_t ld, int64_t inner, int kind, bool strided, bool padded)
{
    const int ch = 16 / fe_size(kind);
    return kind != FGNN_F32 && kind != FGNN_E4M3 && fgnn_aligned16(p) && ld % ch == 0 && (padded ? ld >= (inner + ch - 1) / ch * ch : inner % ch == 0) && inner > 0
        && gm_near(ld * fe_size(kind), strided);
}

template <int KIND, typename E>
static void gm_launch_any(const GemmP &p, bool qs, bool ps, hipStream_t st)
{
    const dim3 g((unsigned)((int64_t)p.tiles_m * p.tiles_n * p.splits)), b(256);
    if constexpr (fe_size_of<KIND> == 1) hipLaunchKernelGGL((gemm_any_kernel<KIND, E, false, false>), g, b, 0, st, p);
    else if (qs) hipLaunchKernelGGL((gemm_any_kernel<KIND, E, true, true>), g, b, 0, st, p);
    else if (ps) hipLaunchKernelGGL((gemm_any_kernel<KIND, E, false, true>), g, b, 0, st, p);
    else hipLaunchKernelGGL((gemm_any_kernel<KIND, E, false, false>), g, b, 0, st, p);
}
template <typename E, typename S>
static void gm_join(const GemmP &p, hipStream_t st)
{
    if (p.splits == 1) return;
    // eight threads a column where it has many parts and there are few columns (256 x 128 of 128 parts 67 / 12 us)
    const int64_t quads = p.m * ((p.n + 3) / 4);
    if (p.splits >= 16 && quads < 256 * 256) hipLaunchKernelGGL((gemm_join_kernel<E, S, 8>), dim3((unsigned)((quads + 31) / 32)), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((gemm_join_kernel<E, S, 1>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, p);
}
template <int KIND, typename E, int TILE, bool FORWARD = false>
static void gm_launch_moved(const GemmP &p, bool qs, bool ps, hipStream_t st)
{
    const dim3 g((unsigned)((int64_t)p.tiles_m * p.tiles_n * p.splits)), b(64 * gm_waves(TILE, TILE));
    const size_t lds = gm_moved_lds(TILE, TILE);
    const LinearEpi<E> f{p.epi};
    if constexpr (fe_size_of<KIND> == 1 || FORWARD) hipLaunchKernelGGL((gemm_moved_kernel<KIND, LinearEpi<E>, false, false, TILE, TILE, 1>), g, b, lds, st, p, f);
    else if (qs) hipLaunchKernelGGL((gemm_moved_kernel<KIND, LinearEpi<E>, true, true, TILE, TILE, 1>), g, b, lds, st, p, f);
    else if (ps) hipLaunchKernelGGL((gemm_moved_kernel<KIND, LinearEpi<E>, false, true, TILE, TILE, 1>), g, b, lds, st, p, f);
    else hipLaunchKernelGGL((gemm_moved_kernel<KIND, LinearEpi<E>, false, false, TILE, TILE, 1>), g, b, lds, st, p, f);
}

// Column tiles of a workgroup of the kernel for few rows: two where every compute unit still gets one, and more than 16 rows make it worth reading x half as
// often (4096 -> 8192 bf16, 32 rows 24 / 18 us, 64 rows 38 / 26; 16 rows 17.0 / 16.8, one row 12.7 / 15.9; 8192 -> 4096 32 rows 24 / 31).
static int gm_rows_ct(int64_t m, int n) { return m > 16 && n >= 32 * gm_units() ? 2 : 1; }
// Whether that kernel is taken.  It reads the rows again for every 16 or 32 columns, where the tiles read them once a 128 and join a cut reduction: us,
// it / tiles, 16 rows 8192 -> 4096 bf16 17.4 / 19.0, 8-bit integers 10.4 / 15.1, 1024 -> 1024 4.1 / 8.0; with 67 MB read again 18.3 / 19.3, with 134 MB 24.2 / 21.3
// and 26.0 / 23.2.  The tiles that convert their operands are slower: with 134 MB 21.4 / 26.4 (8-bit floats), 268 MB 47 / 54 and 51 / 53, 536 MB 75 / 56 (fp32).
static bool gm_few(const GemmP &p, int kind, bool moved)
{
    const int64_t again = (p.m + 15) / 16 * p.k * p.n * fe_size(kind) / gm_rows_ct(p.m, p.n);
    if (!gm_launches(p.n / 16 + 1, 64 * GR_WAVES)) return false;
    return p.m <= 16 || (p.m <= 64 && again <= (moved ? 100000000 : 300000000));
}
template <int KIND, typename E>
static void gm_launch_rows(const GemmP &p, hipStream_t st)
{
    const int64_t blocks = (p.k * GemmKind<KIND>::size + 255) / 256;
    auto go = [&]<int RT, int CT>() {
        // eight waves a compute unit, and as many a workgroup as that takes (4096 -> 8192, 512 groups, 4 / 8 waves 12.7 / 13.5 us; 8192 -> 4096 in 8 bits, 256
        // groups, 8.7 / 8.4)
        const int64_t groups = (p.n + 16 * CT - 1) / (16 * CT);
        const int waves = (int)std::max<int64_t>(1, std::min<int64_t>(2 * groups > 3 * gm_units() ? 4 : 8, blocks));
        hipLaunchKernelGGL((gemm_rows_kernel<KIND, E, RT, CT>), dim3((unsigned)groups), dim3(64 * waves), (size_t)waves * RT * CT * 1024, st, p);
    };
    const int ct = gm_rows_ct(p.m, p.n);
    if (p.m <= 16) go.template operator()<1, 1>();
    else if (p.m <= 32 && ct == 1) go.template operator()<2, 1>();
    else if (p.m <= 32) go.template operator()<2, 2>();
    else if (ct == 1) go.template operator()<4, 1>();
    else go.template operator()<4, 2>();
}

// Tiles of 256 x 256 where there are enough of them for every compute unit, of 128 x 128 else.
static int gm_tile_for(int64_t m, int n)
{
    return ((m + 255) / 256) * ((n + 255) / 256) >= gm_units() ? 256 : 128;
}

static size_t gm_part_bytes(const GemmP &p) { return p.splits > 1 ? (size_t)p.splits * p.m * p.n * sizeof(float) : 0; }
// Partial sums and operands laid out anew; loose: an operand may not be movable as it lies.
static size_t gm_workspace(int64_t m, int n, int64_t k, int kind, bool qs, bool ps, bool loose)
{
    if (m <= 16 && !qs && !ps) return 0;
    GemmP p{};
    p.m = m; p.n = n; p.k = k;
    gm_cut(&p, 128, kind, false);          // (what moves its operands is cut into fewer)
    size_t bytes = fgnn_align256(gm_part_bytes(p));
    if (loose && gm_packs(m, n, k, kind, qs, ps)) bytes += (qs ? gm_packed_bytes(k, m) : gm_packed_bytes(m, k)) + (ps ? gm_packed_bytes(k, n) : gm_packed_bytes(n, k)) + 256;
    return bytes;
}

// D [m, n] of type `type` from operands of kind `kind`; qs: Q is strided along the reduction (and P then too).
static int gm_product(const char *who, GemmP p, int kind, int type, bool qs, bool ps, bool q_padded, void *workspace, size_t workspace_bytes, hipStream_t st)
{
    FGNN_REQUIRE(p.n <= GM_MOST_COLUMNS, FGNN_ERR_LIMIT, "%s: %d columns", who, p.n);
    if (p.m == 0 || p.n == 0) return 0;
    const int64_t inner_q = qs ? p.m : p.k, inner_p = ps ? p.n : p.k;
    const bool q_moves = p.k > 0 && gm_movable(p.q, p.ldq, inner_q, kind, qs, q_padded), p_moves = p.k > 0 && gm_movable(p.p, p.ldp, inner_p, kind, ps, false);
    bool moved = q_moves && p_moves;
    p.rows_q = qs ? (p.m + 7) / 8 * 8 : p.m;                   // (strided operands hold whole chunks of rows, or are made to)
    p.rows_p = ps ? (p.n + 7) / 8 * 8 : p.n;
    if (!moved && p.k > 0 && gm_packs(p.m, p.n, p.k, kind, qs, ps) && !(!qs && !ps && gm_few(p, kind, false))) {
        const int64_t outer_q = qs ? p.k : p.m, outer_p = ps ? p.k : p.n;
        const size_t bytes_q = q_moves ? 0 : gm_packed_bytes(outer_q, inner_q), bytes_p = p_moves ? 0 : gm_packed_bytes(outer_p, inner_p);
        char *to = (char *)(((uintptr_t)workspace + 255) & ~(uintptr_t)255), *after = to + bytes_q + bytes_p;
        gm_cut(&p, gm_tile_for(p.m, p.n), kind, true);
        // (a caller who did not say that an operand may be loose has brought no room for it: then through registers)
        if (workspace && (size_t)(after - (char *)workspace) + gm_part_bytes(p) <= workspace_bytes) {
            if (!q_moves) {
                gm_pack(p.q, p.ldq, outer_q, (int)inner_q, to, kind == FGNN_E4M3, st);
                p.q = to;
                p.ldq = (inner_q + 7) / 8 * 8;
            }
            if (!p_moves) {
                gm_pack(p.p, p.ldp, outer_p, (int)inner_p, to + bytes_q, kind == FGNN_E4M3, st);
                p.p = to + bytes_q;
                p.ldp = (inner_p + 7) / 8 * 8;
            }
            workspace_bytes -= (size_t)(after - (char *)workspace);
            workspace = after;
            if (kind == FGNN_E4M3) kind = FGNN_F16;
            moved = true;
        }
    }
    const bool few = !qs && !ps && gm_few(p, kind, moved);
    const int tile = moved ? gm_tile_for(p.m, p.n) : 128;
    gm_cut(&p, tile, kind, moved);
    if (few) p.splits = 1;
    FGNN_REQUIRE(few || gm_launches((p.m + tile - 1) / tile * p.tiles_n * p.splits, tile == 256 ? 512 : 256), FGNN_ERR_LIMIT, "%s: more tiles than a launch takes", who);
    FGNN_REQUIRE(p.splits == 1 || (workspace && workspace_bytes >= gm_part_bytes(p)), FGNN_ERR_WORKSPACE, "%s: workspace of %zu bytes", who,
                 workspace_bytes);
    p.part = workspace;
    p.epi.m = p.m; p.epi.n = p.n;
    auto launch = [&]<int KIND, typename E>() {
        if (few) return gm_launch_rows<KIND, E>(p, st);
        if constexpr (KIND != FGNN_F32 && KIND != FGNN_E4M3) {
            if (moved && tile == 256) gm_launch_moved<KIND, E, 256>(p, qs, ps, st);
            else if (moved) gm_launch_moved<KIND, E, 128>(p, qs, ps, st);
            else gm_launch_any<KIND, E>(p, qs, ps, st);
        } else gm_launch_any<KIND, E>(p, qs, ps, st);
        gm_join<E, std::conditional_t<KIND == FGNN_I8, int, float>>(p, st);
    };
    // 8-bit floats as fp16: forward products of moved operands alone
    auto launch_widened = [&]<typename E>() {
        if (tile == 256) gm_launch_moved<FGNN_F16, E, 256, true>(p, false, false, st);
        else gm_launch_moved<FGNN_F16, E, 128, true>(p, false, false, st);
        gm_join<E, float>(p, st);
    };
    if (kind == FGNN_F32) launch.template operator()<FGNN_F32, float>();
    else if (kind == FGNN_BF16) launch.template operator()<FGNN_BF16, __bf16>();
    else if (kind == FGNN_F16 && type == FGNN_F16) launch.template operator()<FGNN_F16, _Float16>();
    else if (kind == FGNN_F16 && type == FGNN_BF16) launch_widened.template operator()<__bf16>();
    else if (kind == FGNN_F16) launch_widened.template operator()<float>();
    else fe_dispatch(type, [&]<typename E>() {
        if (kind == FGNN_I8) launch.template operator()<FGNN_I8, E>();
        else launch.template operator()<FGNN_E4M3, E>();
    });
    return fgnn_launch_status(who);
}

static int gm_check_epilogue(const char *who, int type, const void *bias, int btype, const void *res, int64_t ldr, int n, int act)
{
    FGNN_REQUIRE(fe_is_float(type) && (!bias || btype == type || btype == FGNN_F32), FGNN_ERR_SHAPE, "%s: element type %d with bias of type %d", who, type, btype);
    FGNN_REQUIRE(act >= GM_NONE && act <= GM_LEAKY, FGNN_ERR_SHAPE, "%s: activation %d", who, act);
    FGNN_REQUIRE(!res || ldr >= n, FGNN_ERR_SHAPE, "%s: residual rows of %lld", who, (long long)ldr);
    return 0;
}

extern "C" size_t fgnn_linear_workspace_bytes(int64_t rows, int n, int k, int kind, int loose)
{
    if (rows < 1 || n < 1 || n > GM_MOST_COLUMNS || k < 0 || kind < FGNN_F32 || kind > FGNN_E4M3) return 0;
    return gm_workspace(rows, n, k, kind, false, false, loose || kind == FGNN_E4M3);
}

extern "C" int fgnn_linear(int64_t rows, int n, int k, int type, const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, int btype,
                           const void *residual, int64_t ldr, int act, float slope, void *z, void *y, void *workspace, size_t workspace_bytes, void *stream)
{
    FGNN_REQUIRE(rows >= 0 && n >= 0 && k >= 0 && ldx >= k && ldw >= k, FGNN_ERR_SHAPE, "fgnn_linear: bad sizes rows=%lld n=%d k=%d ldx=%lld ldw=%lld",
                 (long long)rows, n, k, (long long)ldx, (long long)ldw);
    const int rc = gm_check_epilogue("fgnn_linear", type, bias, btype, residual, ldr, n, act);
    if (rc) return rc;
    FGNN_REQUIRE(rows == 0 || n == 0 || (y && (k == 0 || (x && weight))), FGNN_ERR_NULL, "fgnn_linear: NULL argument");
    GemmP p{};
    p.m = rows; p.n = n; p.k = k; p.q = x; p.ldq = ldx; p.p = weight; p.ldp = ldw;
    p.epi.bias = bias; p.epi.btype = btype; p.epi.res = residual; p.epi.ldr = ldr; p.epi.act = act; p.epi.slope = slope; p.epi.z = z; p.epi.y = y;
    return gm_product("fgnn_linear", p, type, type, false, false, false, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int fgnn_linear_q8(int64_t rows, int n, int k, int eight, int type, const void *q, int64_t ldq, const float *scale, const void *weight, int64_t ldw,
                              const float *weight_scale, const void *bias, int btype, const void *residual, int64_t ldr, int act, float slope, void *y,
                              void *workspace, size_t workspace_bytes, void *stream)
{
    FGNN_REQUIRE(rows >= 0 && n >= 0 && k >= 0 && ldq >= k && ldw >= k, FGNN_ERR_SHAPE, "fgnn_linear_q8: bad sizes rows=%lld n=%d k=%d ldq=%lld ldw=%lld",
                 (long long)rows, n, k, (long long)ldq, (long long)ldw);
    FGNN_REQUIRE(fe_is_eight(eight), FGNN_ERR_SHAPE, "fgnn_linear_q8: operand type %d", eight);
    FGNN_REQUIRE(eight != FGNN_I8 || k <= 131071, FGNN_ERR_LIMIT, "fgnn_linear_q8: sums of %d products of 8-bit integers do not fit 32 bits", k);
    const int rc = gm_check_epilogue("fgnn_linear_q8", type, bias, btype, residual, ldr, n, act);
    if (rc) return rc;
    FGNN_REQUIRE(rows == 0 || n == 0 || (y && scale && weight_scale && (k == 0 || (q && weight))), FGNN_ERR_NULL, "fgnn_linear_q8: NULL argument");
    GemmP p{};
    p.m = rows; p.n = n; p.k = k; p.q = q; p.ldq = ldq; p.p = weight; p.ldp = ldw;
    p.epi.sx = scale; p.epi.sw = weight_scale;
    p.epi.bias = bias; p.epi.btype = btype; p.epi.res = residual; p.epi.ldr = ldr; p.epi.act = act; p.epi.slope = slope; p.epi.y = y;
    return gm_product("fgnn_linear_q8", p, eight, type, false, false, false, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int fgnn_linear_dx(int64_t rows, int n, int k, int type, const void *dz, int64_t ldz, int padded, const void *weight, int64_t ldw, void *dx, void *workspace,
                              size_t workspace_bytes, void *stream)
{
    FGNN_REQUIRE(rows >= 0 && n >= 0 && k >= 0 && ldz >= n && ldw >= k && fe_is_float(type), FGNN_ERR_SHAPE, "fgnn_linear_dx: bad sizes rows=%lld n=%d k=%d ldz=%lld ldw=%lld type=%d",
                 (long long)rows, n, k, (long long)ldz, (long long)ldw, type);
    FGNN_REQUIRE(rows == 0 || k == 0 || (dx && (n == 0 || (dz && weight))), FGNN_ERR_NULL, "fgnn_linear_dx: NULL argument");
    GemmP p{};
    p.m = rows; p.n = k; p.k = n; p.q = dz; p.ldq = ldz; p.p = weight; p.ldp = ldw;
    p.epi.y = dx;
    return gm_product("fgnn_linear_dx", p, type, type, false, true, padded != 0, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int fgnn_linear_dw(int64_t rows, int n, int k, int type, const void *dz, int64_t ldz, int padded, const void *x, int64_t ldx, void *dw, void *workspace,
                              size_t workspace_bytes, void *stream)
{
    FGNN_REQUIRE(rows >= 0 && n >= 0 && k >= 0 && ldz >= n && ldx >= k && fe_is_float(type), FGNN_ERR_SHAPE, "fgnn_linear_dw: bad sizes rows=%lld n=%d k=%d ldz=%lld ldx=%lld type=%d",
                 (long long)rows, n, k, (long long)ldz, (long long)ldx, type);
    FGNN_REQUIRE(n == 0 || k == 0 || (dw && (rows == 0 || (dz && x))), FGNN_ERR_NULL, "fgnn_linear_dw: NULL argument");
    GemmP p{};
    p.m = n; p.n = k; p.k = rows; p.q = dz; p.ldq = ldz; p.p = x; p.ldp = ldx;
    p.epi.y = dw;
    return gm_product("fgnn_linear_dw", p, type, type, true, true, padded != 0, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" size_t fgnn_linear_backward_workspace_bytes(int64_t rows, int n, int k, int type, int loose)
{
    if (rows < 1 || n < 1 || k < 1 || k > GM_MOST_COLUMNS || !fe_is_float(type)) return 0;
    return std::max(gm_workspace(rows, k, n, type, false, true, loose), gm_workspace(n, k, rows, type, true, true, loose));
}

// ------------------------------------------------------------------------------------------------ slope and column sums
// dz = gy act'(z) and its column sums in one pass: bound by memory.  A workgroup takes a strip of columns (TX 16-byte vectors) and every grid.y-th batch of
// 256 / TX rows; the sums of its rows go to memory as one row of partial sums, added up in a fixed order afterwards.
struct SlopeP {
    int64_t rows; int n;
    const void *gy; int64_t ldg; const void *z;
    int act; float slope;
    void *dz; int64_t ldz;                  // ldz: n, or more with zeros behind n; NULL: not wanted
    float *part;                            // [grid.y][n]; NULL: not wanted
};
template <typename E, int TX>
__global__ __launch_bounds__(256) void linear_slope_kernel(SlopeP p)
{
    constexpr int V = fe_width<E>, TY = 256 / TX;
    __shared__ float sums[TY > 1 ? TY : 1][TX * V];
    const int tx = (int)threadIdx.x % TX, ty = (int)threadIdx.x / TX, c = ((int)blockIdx.x * TX + tx) * V, count = p.n - c;
    float sum[V] = {};
    if (count > 0) {
        for (int64_t row = (int64_t)blockIdx.y * TY + ty; row < p.rows; row += (int64_t)gridDim.y * TY) {
            float g[V];
            gm_load<E, V>(g, (const E *)p.gy + row * p.ldg + c, count);
            if (p.act) {
                float z[V];
                gm_load<E, V>(z, (const E *)p.z + row * p.n + c, count);
                gm_act_slope(g, z, p.act, p.slope);
            }
            if (p.dz) gm_store<E, V>(g, (E *)p.dz + row * p.ldz + c, p.ldz == p.n ? count : V);          // (values past a row's end were read as zeros)
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] += g[i];
        }
    }
    if (!p.part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) sums[ty][tx * V + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < TX * V; i += 256) {
        const int col = (int)blockIdx.x * TX * V + i;
        if (col >= p.n) break;
        float v = 0.f;
#pragma unroll
        for (int t = 0; t < TY; ++t) v += sums[t][i];
        p.part[(int64_t)blockIdx.y * p.n + col] = v;
    }
}

static int sl_width(int n, int type)
{
    const int vectors = (n + 16 / fe_size(type) - 1) / (16 / fe_size(type));
    return vectors <= 8 ? 8 : vectors <= 32 ? 32 : vectors <= 64 ? 64 : 256;
}
static dim3 sl_grid(int64_t rows, int n, int type)
{
    const int tx = sl_width(n, type), v = 16 / fe_size(type), strips = (n + tx * v - 1) / (tx * v), high = 256 / tx;
    const int64_t most = std::max(1, 4 * gm_units() / strips);
    return dim3((unsigned)strips, (unsigned)std::max<int64_t>(1, std::min<int64_t>((rows + high - 1) / high, most)));
}

extern "C" size_t fgnn_linear_slope_workspace_bytes(int64_t rows, int n, int type)
{
    if (rows < 1 || n < 1 || n > GM_MOST_COLUMNS || !fe_is_float(type)) return 0;
    return (size_t)sl_grid(rows, n, type).y * n * sizeof(float);
}

extern "C" int fgnn_linear_slope(int64_t rows, int n, int type, const void *gy, int64_t ldg, const void *z, int act, float slope, void *dz, int64_t ldz, void *dbias, int btype,
                                 void *workspace, size_t workspace_bytes, void *stream)
{
    FGNN_REQUIRE(rows >= 0 && n >= 1 && ldg >= n && fe_is_float(type) && act >= GM_NONE && act <= GM_LEAKY, FGNN_ERR_SHAPE,
                 "fgnn_linear_slope: bad sizes rows=%lld n=%d ldg=%lld type=%d act=%d", (long long)rows, n, (long long)ldg, type, act);
    FGNN_REQUIRE(n <= GM_MOST_COLUMNS, FGNN_ERR_LIMIT, "fgnn_linear_slope: %d columns", n);
    FGNN_REQUIRE(!dbias || btype == type || btype == FGNN_F32, FGNN_ERR_SHAPE, "fgnn_linear_slope: bias of type %d", btype);
    const int width = fe_is_float(type) ? 16 / fe_size(type) : 1;
    FGNN_REQUIRE(!dz || ldz == n || ldz == (n + width - 1) / width * width, FGNN_ERR_SHAPE, "fgnn_linear_slope: rows of %lld for %d columns", (long long)ldz, n);
    FGNN_REQUIRE(rows == 0 || (gy && (act == GM_NONE || z)), FGNN_ERR_NULL, "fgnn_linear_slope: NULL argument");
    FGNN_REQUIRE(!dbias || rows == 0 || (workspace && workspace_bytes >= fgnn_linear_slope_workspace_bytes(rows, n, type)), FGNN_ERR_WORKSPACE,
                 "fgnn_linear_slope: workspace of %zu bytes", workspace_bytes);
    hipStream_t st = (hipStream_t)stream;
    int parts = 0;
    if (rows > 0 && (dz || dbias)) {
        const dim3 g = sl_grid(rows, n, type);
        parts = (int)g.y;
        SlopeP p{rows, n, gy, ldg, z, act, slope, dz, ldz, dbias ? (float *)workspace : nullptr};
        fe_dispatch(type, [&]<typename E>() {
            switch (sl_width(n, type)) {
            case 8: hipLaunchKernelGGL((linear_slope_kernel<E, 8>), g, dim3(256), 0, st, p); break;
            case 32: hipLaunchKernelGGL((linear_slope_kernel<E, 32>), g, dim3(256), 0, st, p); break;
            case 64: hipLaunchKernelGGL((linear_slope_kernel<E, 64>), g, dim3(256), 0, st, p); break;
            default: hipLaunchKernelGGL((linear_slope_kernel<E, 256>), g, dim3(256), 0, st, p);
            }
        });
        const int rc = fgnn_launch_status("linear_slope_kernel");
        if (rc) return rc;
    }
    return dbias ? fgnn_sum_parts((const float *)workspace, parts, n, dbias, btype, st) : 0;
}
