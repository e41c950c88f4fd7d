"""Linear maps with bias, activation and residual in the epilogue, their gradients, and the same over operands in 8 bits, against float64."""
import math

import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.operators import linear_act, linear_q8, quantize_rows

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(UNIT)
# rows, k, n: single rows and columns, either side of tiles and slabs, odd widths (rows of 16-bit values at odd addresses), long reductions over small
# results and large results over short ones
SIZES = [(1, 1, 1), (1, 64, 256), (3, 7, 5), (16, 128, 64), (17, 129, 65), (64, 31, 130), (127, 256, 128), (129, 100, 257), (300, 602, 41), (33, 1433, 16),
         (1000, 64, 64), (5, 5000, 48), (2500, 33, 7), (513, 384, 512), (1, 4097, 300), (40, 2048, 1030)]


def act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "leaky_relu":
        return torch.where(z > 0, z, 0.2 * z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    return z * torch.sigmoid(z) if name == "silu" else z


def allowance(dtype, ref, terms, extra=0.0):
    """One rounding of the result to its type; sums in 32 bits: 16 roundings of the sum of magnitudes `terms` (a long sum is made of shorter ones;
    fp32's three parts leave 2^-23 of a product); `extra`: what operands rounded to the type on the way add."""
    return 1.01 * UNIT[dtype] * ref.abs() + 16 * 2.0 ** -24 * terms + extra + (2.0 ** -24 if dtype is torch.float16 else 0)


def within(got, ref, tol, what):
    got, ref, tol = got.detach().double().cpu(), ref.detach().cpu(), tol.detach().cpu()
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), "%s: %d of %d outside, worst %.3g of the allowance" % (what, int(bad.sum()), bad.numel(), float(((got - ref).abs() / tol).max()))


def operands(rows, k, n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + rows + 7 * k + 11 * n)
    x, w, b, r, gy = (torch.randn(s, generator=g) for s in ((rows, k), (n, k), (n,), (rows, n), (rows, n)))
    return [t.to(dtype) for t in (x, w * k ** -0.5, b, r, gy)]


def check_all(rows, k, n, dtype, name, with_bias=True, with_residual=True):
    x, w, b, r, gy = operands(rows, k, n, dtype)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b, r)]
    y = linear_act(leaves[0], leaves[1], leaves[2] if with_bias else None, residual=leaves[3] if with_residual else None, activation=name)
    y.backward(gy.cuda())
    xd, wd, bd, rd, gyd = (t.double() for t in (x, w, b, r, gy))
    z = (xd @ wd.t() + (bd if with_bias else 0)).requires_grad_(True)
    a = act(z, name)
    ref = a + (rd if with_residual else 0)
    magnitude = xd.abs() @ wd.abs().t() + bd.abs() + rd.abs()
    # an activation's slope is at most 1.13; z's own size counts for the exponentials behind it
    within(y, ref, allowance(dtype, ref, 2 * magnitude + z.detach().abs()), "y")
    (dz,) = torch.autograd.grad(a, z, gyd)
    dz = dz.detach()
    # dz is formed from z in the rows' type and rounded to it; where z lies within its own rounding of zero a relu's slope may be the other one
    unit, zd = UNIT[dtype], z.detach()
    off = 1.01 * unit * dz.abs() + 16 * 2.0 ** -24 * gyd.abs() if name or dtype is torch.float32 else torch.zeros_like(dz)
    if name in ("gelu", "silu"):
        off = off + gyd.abs() * (0.8 * unit * zd.abs() + 16 * 2.0 ** -24 * (1 + magnitude))        # |act''| < 0.8
    if name in ("relu", "leaky_relu"):
        off = off + gyd.abs() * (zd.abs() <= 16 * 2.0 ** -24 * magnitude + (2.0 ** -24 if dtype is torch.float16 else 0))
    dx, dw = dz @ wd, dz.t() @ xd
    within(leaves[0].grad, dx, allowance(dtype, dx, dz.abs() @ wd.abs(), off @ wd.abs()), "dx")
    within(leaves[1].grad, dw, allowance(dtype, dw, dz.abs().t() @ xd.abs(), off.t() @ xd.abs()), "dw")
    if with_bias:
        db = dz.sum(0)
        within(leaves[2].grad, db, allowance(dtype, db, dz.abs().sum(0), off.sum(0)), "db")
    if with_residual:
        assert torch.equal(leaves[3].grad, gy.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_sizes(dtype, size):
    check_all(*size, dtype, "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", [None, "relu", "gelu", "silu", "leaky_relu"])
@pytest.mark.parametrize("rows", [2, 200])
def test_activations(dtype, name, rows):
    for with_bias, with_residual in ((True, True), (False, True), (True, False), (False, False)):
        check_all(rows, 96, 80, dtype, name, with_bias, with_residual)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_larger_products(dtype):
    check_all(1030, 1100, 1290, dtype, "silu")
    check_all(20011, 128, 256, dtype, "relu")
    check_all(2048, 1024, 2048, dtype, None)
    # rows at odd addresses, with and without an activation in between
    check_all(1501, 1003, 1201, dtype, "gelu")
    check_all(1501, 1003, 1201, dtype, None)
    check_all(1504, 1001, 1208, dtype, "relu")
    check_all(1501, 1008, 1204, dtype, None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65])
def test_few_rows(dtype, rows):
    # either side of every number of row tiles; columns in one tile and two a workgroup; reductions shorter and longer than a block of every wave
    for k, n in ((20, 40), (700, 100), (2100, 33), (130, 8200)):
        check_all(rows, k, n, dtype, "relu")


@pytest.mark.gpu
def test_gradient_against_differences():
    x, w, b, r, gy = operands(9, 12, 10, torch.float32)
    for name in (None, "gelu", "silu", "leaky_relu"):
        leaves = [t.cuda().requires_grad_(True) for t in (x, w, b, r)]
        linear_act(*leaves[:3], residual=leaves[3], activation=name).backward(gy.cuda())
        base = [t.double() for t in (x, w, b, r)]

        def value(t):
            return float(((act(t[0] @ t[1].t() + t[2], name) + t[3]) * gy.double()).sum())
        for which, leaf in enumerate(leaves):
            for at in range(0, leaf.numel(), 5):
                ends = []
                for sign in (1, -1):
                    moved = [t.clone() for t in base]
                    moved[which].view(-1)[at] += sign * 1e-6
                    ends.append(value(moved))
                assert abs(float(leaf.grad.view(-1)[at]) - (ends[0] - ends[1]) / 2e-6) < 2e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_types_of_bias(dtype):
    g = torch.Generator().manual_seed(1)
    wide = torch.randn(70, 150, generator=g).to(dtype).cuda()
    x, w, r = wide[:, 3:100], wide[:37, 5:102], wide[:, 101:138]
    b = torch.randn(37, generator=g).cuda()                    # fp32 beside any rows
    z = x.double() @ w.double().t() + b.double()
    ref = act(z, "silu") + r.double()
    tol = allowance(dtype, ref, 2 * (x.double().abs() @ w.double().abs().t() + b.double().abs() + r.double().abs()))
    within(linear_act(x, w, b, residual=r, activation="silu"), ref, tol, "strided rows")
    within(linear_act(x.t().contiguous().t(), w.t().contiguous().t(), b, residual=r, activation="silu"), ref, tol, "strided columns")
    within(linear_act(x.reshape(7, 10, 97), w, b, residual=r.reshape(7, 10, 37), activation="silu").reshape(70, 37), ref, tol, "three dimensions")
    one = linear_act(x[0], w, b, residual=r[0], activation="silu")
    assert one.shape == (37,)
    within(one, ref[0], tol[0], "a vector")
    # a bias of 32 bits gets its gradient in 32 bits, summed before anything is rounded
    bl = b.clone().requires_grad_(True)
    gy = torch.randn(70, 37, generator=g).to(dtype).cuda()
    (db,) = torch.autograd.grad(linear_act(x, w, bl), bl, gy)
    assert db.dtype is torch.float32
    within(db, gy.double().sum(0), 16 * 2.0 ** -24 * gy.double().abs().sum(0), "db")
    # an expanded gradient, as of a sum
    xl = x.clone().requires_grad_(True)
    linear_act(xl, w, b).sum().backward()
    dx = w.double().sum(0).expand(70, 97)
    within(xl.grad, dx, allowance(dtype, dx, w.double().abs().sum(0).expand(70, 97)), "gradient of a sum")
    # one operand only
    for which in range(4):
        leaves = [t.clone() for t in (x, w, b, r)]
        leaves[which].requires_grad_(True)
        linear_act(*leaves[:3], residual=leaves[3], activation="relu").sum().backward()
        assert leaves[which].grad.shape == leaves[which].shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_sum_and_nothing_to_write(dtype):
    w0, b, r = torch.empty(6, 0, dtype=dtype).cuda(), torch.randn(6).to(dtype).cuda(), torch.randn(4, 6).to(dtype).cuda()
    got = linear_act(torch.empty(4, 0, dtype=dtype).cuda(), w0, b, residual=r, activation="relu")
    assert torch.equal(got, (b.float().clamp_min(0) + r.float()).to(dtype))
    x, w, bl = (t.requires_grad_(True) for t in (torch.empty(0, 8, dtype=dtype).cuda(), torch.randn(6, 8).to(dtype).cuda(), b.clone()))
    y = linear_act(x, w, bl, activation="gelu")
    assert y.shape == (0, 6)
    y.sum().backward()
    assert x.grad.shape == (0, 8) and (w.grad == 0).all() and (bl.grad == 0).all()
    assert linear_act(torch.randn(3, 8).to(dtype).cuda(), torch.empty(0, 8, dtype=dtype).cuda()).shape == (3, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(5, 40, 33), (200, 64, 128), (700, 700, 300)])
def test_infinities_and_nan_stay_in_their_rows(dtype, size):
    x, w, b, r, _ = operands(*size, dtype)
    clean = linear_act(x.cuda(), w.cuda(), b.cuda())
    x[1, 3], x[3, 0], x[4, 7] = float("inf"), float("nan"), float("-inf")
    w[2, 7] = 0.5
    got = linear_act(x.cuda(), w.cuda(), b.cuda()).cpu()
    ref = (x.double() @ w.double().t() + b.double())
    keep = [i for i in range(size[0]) if i not in (1, 3, 4)]
    other = [j for j in range(size[2]) if j != 2]
    assert torch.equal(got[keep][:, other], clean.cpu()[keep][:, other])
    assert got[3].isnan().all()
    assert torch.equal(got[1].double(), ref[1]) and torch.equal(got[4].double(), ref[4])
    # values near the type's largest: products of them reach infinity as they do in 32 bits, sums do not lose finite ones
    big = torch.full((2, 8), 3e38 if dtype is not torch.float16 else 6e4, dtype=dtype).cuda()
    eye = torch.eye(8, dtype=dtype).cuda()
    assert torch.equal(linear_act(big, eye), big)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES + [(700, 512, 384), (1100, 1010, 1030), (1500, 1024, 1024)])
def test_eight_bits(eight, dtype, size):
    rows, k, n = size
    x, w, b, r, _ = operands(rows, k, n, torch.float32)
    b, r = b.to(dtype), r.to(dtype)
    q, s = quantize_rows(x.cuda(), eight)
    wq, ws = quantize_rows(w.cuda(), eight)
    for name, bias, residual in ((None, b, r), ("silu", b, None), ("gelu", None, r), ("relu", b.float(), None)):
        y = linear_q8(q, s, wq, ws, None if bias is None else bias.cuda(), residual=None if residual is None else residual.cuda(), activation=name, dtype=dtype)
        xd, wd = q.cpu().double() * s.cpu().double()[:, None], wq.cpu().double() * ws.cpu().double()[:, None]
        z = xd @ wd.t() + (0 if bias is None else bias.double())
        ref = act(z, name) + (0 if residual is None else residual.double())
        magnitude = xd.abs() @ wd.abs().t() + b.double().abs() + r.double().abs()
        within(y, ref, allowance(dtype, ref, 2 * magnitude + z.abs()), "y")
    if eight is torch.int8:
        # the sums themselves are exact
        one = torch.ones(rows).cuda(), torch.ones(n).cuda()
        got = linear_q8(q, one[0], wq, one[1], dtype=torch.float32)
        assert torch.equal(got.cpu(), (q.cpu().double() @ wq.cpu().double().t()).float()) or k > 1000


@pytest.mark.gpu
def test_eight_bit_strides_and_empty_rows():
    wide = torch.randint(-127, 128, (40, 300), dtype=torch.int8).cuda()
    q, wq = wide[:, 1:200], wide[:30, 3:202]
    s, ws = torch.rand(40).cuda(), torch.rand(30).cuda()
    ref = (q.double() * s.double()[:, None]) @ (wq.double() * ws.double()[:, None]).t()
    tol = allowance(torch.bfloat16, ref, (q.double().abs() * s.double()[:, None]) @ (wq.double().abs() * ws.double()[:, None]).t())
    within(linear_q8(q, s, wq, ws), ref, tol, "strided")
    assert linear_q8(q[:0], s[:0], wq, ws).shape == (0, 30)
    # rows of zeros have scale 0, a row without a finite scale is NaN
    s[2], s[5] = 0, float("nan")
    got = linear_q8(q, s, wq, ws)
    assert (got[2] == 0).all() and got[5].isnan().all() and torch.isfinite(got[6:]).all()


@pytest.mark.gpu
def test_other_streams_and_one_order_of_sums():
    x, w, b, r, gy = (t.cuda() for t in operands(3000, 200, 72, torch.bfloat16))
    ref = linear_act(x, w, b, residual=r, activation="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_act(x, w, b, residual=r, activation="gelu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    grads = []
    for _ in range(3):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        linear_act(*leaves, activation="gelu").backward(gy)
        grads.append([t.grad for t in leaves])
    assert all(torch.equal(a, c) for other in grads[1:] for a, c in zip(grads[0], other))


def test_refusals():
    x, w = torch.randn(4, 8), torch.randn(6, 8)
    with pytest.raises(_lib.FgnnError):
        linear_act(x, w)
    with pytest.raises(_lib.FgnnError):
        linear_act(x, w, activation="tanh")
    l, p = _lib.lib(), 256
    assert l.fgnn_linear(2, 6, 8, 0, p, 7, p, 8, None, 0, None, 0, 0, 0.0, None, p, None, 0, None) == -2         # row stride below the columns
    assert l.fgnn_linear(2, 6, 8, 3, p, 8, p, 8, None, 0, None, 0, 0, 0.0, None, p, None, 0, None) == -2         # 8-bit rows
    assert l.fgnn_linear(2, 6, 8, 1, p, 8, p, 8, p, 2, None, 0, 0, 0.0, None, p, None, 0, None) == -2            # bias of the other 16-bit type
    assert l.fgnn_linear(2, 6, 8, 1, p, 8, p, 8, None, 0, p, 5, 0, 0.0, None, p, None, 0, None) == -2            # residual's row stride
    assert l.fgnn_linear(2, 6, 8, 1, p, 8, p, 8, None, 0, None, 0, 5, 0.0, None, p, None, 0, None) == -2         # no such activation
    assert l.fgnn_linear(2, 6, 8, 1, p, 8, None, 8, None, 0, None, 0, 0, 0.0, None, p, None, 0, None) == -1
    assert l.fgnn_linear_q8(2, 6, 131073, 3, 1, p, 131073, p, p, 131073, p, None, 1, None, 0, 0, 0.0, p, None, 0, None) == -4
    assert l.fgnn_linear_q8(2, 6, 8, 1, 1, p, 8, p, p, 8, p, None, 1, None, 0, 0, 0.0, p, None, 0, None) == -2
    assert l.fgnn_linear_slope(2, 6, 0, p, 6, p, 1, 0.0, p, 7, None, 0, None, 0, None) == -2                     # rows of dz neither n nor whole 16 bytes
    assert l.fgnn_linear_slope(2, 6, 0, p, 6, None, 1, 0.0, p, 6, None, 0, None, 0, None) == -1                     # an activation without its argument
    assert l.fgnn_linear_slope(2, 6, 0, p, 6, p, 1, 0.0, p, 6, p, 0, None, 0, None) == -5                           # no workspace for the sums
    big = l.fgnn_linear_workspace_bytes(100, 16, 100000, 1, 0)
    assert big > 0 and l.fgnn_linear(100, 16, 100000, 1, p, 100000, p, 100000, None, 0, None, 0, 0, 0.0, None, p, p, big - 4, None) == -5


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, w, b = torch.randn(4, 8).cuda(), torch.randn(6, 8).cuda(), torch.randn(6).cuda()
    q, s = quantize_rows(x)
    wq, ws = quantize_rows(w)
    for bad in (lambda: linear_act(x, w[:, :7]), lambda: linear_act(x, w.half()), lambda: linear_act(x.double(), w.double()), lambda: linear_act(x, w, b[:5]),
                lambda: linear_act(x, w, b.half()), lambda: linear_act(x, w, b, residual=x), lambda: linear_act(x, w, b.cpu()),
                lambda: linear_act(x, w, residual=torch.randn(4, 6).cuda().half()), lambda: linear_act(x, w[0]),
                lambda: linear_q8(q, s, wq.float(), ws), lambda: linear_q8(q, s[:3], wq, ws), lambda: linear_q8(q, s.half(), wq, ws),
                lambda: linear_q8(q, s, wq, ws, dtype=torch.float64), lambda: linear_q8(q, s, wq, ws, b.half()), lambda: linear_q8(q, s, wq[:, :4], ws)):
        with pytest.raises(_lib.FgnnError):
            bad()


@pytest.mark.gpu
def test_second_order_gradients_are_refused():
    x, w = torch.randn(4, 8).cuda().requires_grad_(True), torch.randn(6, 8).cuda().requires_grad_(True)
    (dx,) = torch.autograd.grad(linear_act(x, w, activation="gelu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second order"):
        dx.sum().backward()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    from ae_mlsys_gnn_amd.operators import rms_norm
    rows, k = 2200003, 1000                                      # 2.2e9 values
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    for part in x.split(200000):
        part.normal_()
    w = torch.randn(24, k, device="cuda").to(torch.bfloat16)
    y = linear_act(x, w)
    picks = torch.tensor([0, 1, 2147483, 2147484, rows - 130, rows - 2, rows - 1], device="cuda")
    z = x[picks].double() @ w.double().t()
    within(y[picks], z, allowance(torch.bfloat16, z, x[picks].double().abs() @ w.double().abs().t()), "rows")
    g = torch.zeros(rows, 24, dtype=torch.bfloat16, device="cuda")
    g[picks] = 1
    wl = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(linear_act(x, wl), wl, g)
    ref = x[picks].double().sum(0).expand(24, k)
    within(dw, ref, allowance(torch.bfloat16, ref, x[picks].double().abs().sum(0).expand(24, k)), "dw")
    n = rms_norm(x)
    assert torch.equal(n[picks], rms_norm(x[picks]))
