"""The dense operators at the ends of their ranges: long rows and row strides, small and large values, sums of integers, what they refuse."""
import glob
import os
import re

import pytest
import torch
from torch.utils.flop_counter import FlopCounterMode

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.layers import ResidualBlock
from ae_mlsys_gnn_amd.operators import linear_act, linear_q8, orthogonalize, quantize_rows, rms_norm, rms_norm_q8
from ae_mlsys_gnn_amd.train.muon import Muon

from .test_linear_gpu import act, allowance, within

F32, BF16, F16, I8, E4M3 = range(5)
CSRC = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")


def test_rows_past_32_bit_offsets_are_not_laid_out_anew():
    # what moves operands has 32-bit offsets in a tile of up to 256 rows: rows of 2^23 bytes and more stay where they are, and need no room to be laid out in
    l = _lib.lib()
    for kind in (BF16, F16, E4M3):
        laid_out = 128 * 4194296 * 2
        assert l.fgnn_linear_workspace_bytes(128, 8, 4194296 - 1, kind, 1) >= laid_out
        assert l.fgnn_linear_workspace_bytes(128, 8, 4194304 + 1, kind, 1) < laid_out
        assert l.fgnn_linear_workspace_bytes(128, 8, 8454665, kind, 1) < laid_out
    # strided ones, of which a tile takes 64 rows: of 2^25 bytes
    assert l.fgnn_linear_backward_workspace_bytes(64, 16777216 - 15, 8, BF16, 1) >= 64 * (16777216 - 16) * 2
    assert l.fgnn_linear_backward_workspace_bytes(64, 16777216 + 1, 8, BF16, 1) < 64 * 16777216 * 2


@pytest.mark.gpu
def test_odd_reduction_past_32_bit_offsets():
    rows, k, n = 128, 8454665, 8
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = torch.empty(n, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    y = linear_act(x, w)
    wd = w.double()
    for i in (0, 1, 63, 125, 126, 127):
        xd = x[i:i + 1].double()
        ref = (xd * wd).sum(-1)
        within(y[i], ref, allowance(torch.bfloat16, ref, (xd * wd).abs().sum(-1)), "row %d" % i)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: without a device nothing is launched")
def test_long_row_strides_need_no_room_that_was_not_asked_for():
    l, p = _lib.lib(), 4096
    # (rows, n, k, row stride of x): aligned 16-bit rows, so far apart that they are not moved as they lie
    for rows, n, k, ldx in ((512, 32000, 4096, 4194304), (300, 32000, 4096, 4194304), (200, 128256, 4096, 8388608), (128, 64, 4194304, 4194304)):
        told = l.fgnn_linear_workspace_bytes(rows, n, k, BF16, 0)
        assert l.fgnn_linear(rows, n, k, BF16, p, ldx, p, k, None, 0, None, 0, 0, 0.0, None, p, p, told, None) not in (0, -5), (rows, n, k)
    # the same by an address that is not said to be loose, and in a gradient
    told = l.fgnn_linear_workspace_bytes(2048, 2048, 1024, BF16, 0)
    assert l.fgnn_linear(2048, 2048, 1024, BF16, p + 2, 1024, p, 1024, None, 0, None, 0, 0, 0.0, None, p, p, told, None) not in (0, -5)
    told = l.fgnn_linear_backward_workspace_bytes(512, 2048, 4096, BF16, 0)
    assert l.fgnn_linear_dw(512, 2048, 4096, BF16, p, 2048, 0, p, 33554432, p, p, told, None) not in (0, -5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_far_apart(dtype):
    # the last of 1024 positions of every sequence, before a wide layer
    rows, k, n, ld = 512, 4096, 1536, 4194304
    g = torch.Generator(device="cuda").manual_seed(1)
    space = torch.empty((rows - 1) * ld + k, dtype=dtype, device="cuda")
    x = space.as_strided((rows, k), (ld, 1))
    x.normal_(generator=g)
    w = torch.empty(n, k, dtype=dtype, device="cuda").normal_(0, k ** -0.5, generator=g)
    gy = torch.empty(rows, n, dtype=dtype, device="cuda").normal_(generator=g)
    xl, wl = x.detach().requires_grad_(True), w.clone().requires_grad_(True)
    assert xl.stride() == (ld, 1)
    y = linear_act(xl, wl)
    dx, dw = torch.autograd.grad(y, (xl, wl), gy)
    xd, wd, gd = x.double(), w.double(), gy.double()
    for got, a, b, what in ((y, xd, wd.t(), "y"), (dx, gd, wd, "dx"), (dw, gd.t(), xd, "dw")):
        b = b.contiguous()
        ref = a @ b
        within(got, ref, allowance(dtype, ref, a.abs() @ b.abs()), what)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(100, 90), (300, 520), (1100, 700)])
def test_planes_of_every_element(dtype, shape):
    # one step with a = 1, b = c = 0 hands X_0 back as its two planes hold it, to 2^-23 of each element; X_0 itself and the result are four roundings in 32 bits
    g = torch.Generator().manual_seed(3)
    m = (1 + torch.rand(shape, generator=g)).to(dtype)
    got = orthogonalize(m.cuda(), steps=1, coefficients=(1.0, 0.0, 0.0)).double().cpu()
    ref = m.double() / (m.double().norm() + 1e-7)
    own = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    assert ((got - ref).abs() <= (2.0 ** -23 + 4 * 2.0 ** -24 + 1.01 * own) * ref.abs() + 2.0 ** -50 + (2.0 ** -25 if dtype is torch.float16 else 0)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 40), (40, 2), (300, 520)])
def test_planes_of_small_elements(shape):
    # one step with a = 1, b = c = 0 hands X_0 back as its two planes hold it: elements of 2^-16 to 2^-32 of the norm beside one that is the norm.  The planes of
    # an X_0 scaled by 2^14 hold 2^-23 of an element, and 2^-36 where that is less; X_0 itself and the result are four roundings in 32 bits
    g = torch.Generator().manual_seed(2)
    m = torch.randn(shape, generator=g) * torch.exp2(-16.0 * (1 + torch.rand(shape, generator=g)))
    m[0, 0] = 1.0
    got = orthogonalize(m.cuda(), steps=1, coefficients=(1.0, 0.0, 0.0)).double().cpu()
    ref = m.double() / (m.double().norm() + 1e-7)
    assert ((got - ref).abs() <= (2.0 ** -23 + 4 * 2.0 ** -24) * ref.abs() + 2.0 ** -50).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1, 64, 64), (1, 61, 33), (40, 128, 96), (40, 129, 97), (300, 128, 256), (300, 129, 257), (1501, 1003, 1201)])
def test_operands_below_fp16s_normal_range(rows, k, n):
    # 1e-5 to 6e-5 lies below 2^-14: as rows, as weights and as gradients, beside values that keep the results within range
    g = torch.Generator().manual_seed(4)

    def small(*shape):
        return ((1e-5 + 5e-5 * torch.rand(shape, generator=g)) * torch.randn(shape, generator=g).sign()).half().cuda()

    def large(*shape):
        return (64 * torch.randn(shape, generator=g)).half().cuda()

    def product(got, a, b, what):
        a, b = a.double(), b.double().contiguous()
        ref = a @ b
        within(got, ref, allowance(torch.float16, ref, a.abs() @ b.abs()), what)

    x, w, gy = small(rows, k), small(n, k), small(rows, n)
    xs, ws = large(rows, k), large(n, k)
    product(linear_act(x, ws), x, ws.t(), "small rows")
    product(linear_act(xs, w), xs, w.t(), "small weights")
    # gradients straight into the products, and by way of an activation's slope (1 here: all that goes into the sums is positive)
    for name in (None, "relu"):
        leaves = (xs.abs() / 64).requires_grad_(True), ws.abs().requires_grad_(True)
        dx, dw = torch.autograd.grad(linear_act(*leaves, activation=name), leaves, gy)
        product(dx, gy, leaves[1].detach(), "dx")
        product(dw, gy.t(), leaves[0].detach(), "dw")


def test_sums_of_8_bit_integers_fit_32_bits():
    # 131,072 products of -128 by -128 are 2^31
    l, p = _lib.lib(), 4096
    assert l.fgnn_linear_q8(2, 6, 131072, I8, BF16, p, 131072, p, p, 131072, p, None, 1, None, 0, 0, 0.0, p, None, 0, None) == -4


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 200])
def test_largest_sums_of_8_bit_integers(rows):
    q, w = (torch.full((n, 131071), -128, dtype=torch.int8, device="cuda") for n in (rows, 20))
    y = linear_q8(q, torch.ones(rows, device="cuda"), w, torch.ones(20, device="cuda"), dtype=torch.float32)
    assert (y == 131071 * 16384).all()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: without a device nothing is launched")
def test_columns_that_32_bits_cannot_count_are_refused():
    # the last tile of columns ends past 2^31
    l, p = _lib.lib(), 4096
    n, most = 2 ** 31 - 100, 2 ** 31 - 4096
    for rows in (1, 100):
        assert l.fgnn_linear(rows, n, 1, BF16, p, 1, p, 1, None, 0, None, 0, 0, 0.0, None, p, None, 0, None) == -4
        assert l.fgnn_linear(rows, most, 1, BF16, p, 1, p, 1, None, 0, None, 0, 0, 0.0, None, p, None, 0, None) != 0
    assert l.fgnn_linear_q8(1, n, 1, I8, BF16, p, 1, p, p, 1, p, None, 1, None, 0, 0, 0.0, p, None, 0, None) == -4
    assert l.fgnn_linear_dx(1, 1, n, BF16, p, 1, 0, p, n, p, None, 0, None) == -4
    assert l.fgnn_linear_dw(1, 1, n, BF16, p, 1, 0, p, n, p, None, 0, None) == -4
    assert l.fgnn_linear_slope(1, n, BF16, p, n, p, 1, 0.0, p, n, None, 0, None, 0, None) == -4


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up: without a device nothing is launched")
def test_more_tiles_than_a_launch_takes_are_refused():
    # 2^24 tiles of 256 threads are 2^32 threads
    l, p = _lib.lib(), 4096
    assert l.fgnn_linear(2 ** 31, 1, 1, BF16, p, 1, p, 1, None, 0, None, 0, 0, 0.0, None, p, None, 0, None) == -4
    assert l.fgnn_linear(2 ** 31 - 128, 1, 1, BF16, p, 1, p, 1, None, 0, None, 0, 0, 0.0, None, p, None, 0, None) not in (0, -4)


@pytest.mark.gpu
def test_a_row_of_many_columns():
    # more columns than a launch of the kernel for few rows, or one of the bias gradient's last sum, has threads for
    n = 2 ** 28 + 40
    x = torch.randn(2, 1).cuda().bfloat16()
    w = torch.randn(n, 1, device="cuda").bfloat16()
    b = torch.zeros(n, device="cuda", requires_grad=True)
    y = linear_act(x, w, b)
    assert torch.equal(y.detach(), (x.float() * w.float().t()).bfloat16())
    (db,) = torch.autograd.grad(y, b, y.detach())
    assert torch.equal(db, y.detach().float().sum(0))


def test_assembly_declares_what_it_writes():
    # a scalar register that an instruction of a statement names as its first operand is among what the statement says it changes
    seen = 0
    for path in glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(CSRC, "*.hip")):
        for body in re.findall(r"\basm(?:\s+volatile)?\s*\((.*?)\);", open(path).read(), flags=re.S):
            parts = re.split(r":(?=(?:[^\"]*\"[^\"]*\")*[^\"]*$)", body)
            seen += 1
            for written in re.findall(r"\bs_\w+\s+(m0|vcc|exec|s\d+)\b", parts[0]):
                assert len(parts) == 4 and '"%s"' % written in parts[3], (os.path.basename(path), written)
    assert seen >= 3


@pytest.mark.gpu
def test_last_sums_of_column_sums():
    # 2^24 beside 63 ones: each part of the sum is exact, and 32 bits would drop every one added to it alone.  Rows are dealt out in turns of 32, so that the
    # ones stand in other parts than the large value
    gy = torch.zeros(2048, 32)
    gy[0] = 2.0 ** 24
    gy[32::32] = 1.0
    b = torch.zeros(32, device="cuda", requires_grad=True)
    x, w = torch.zeros(2048, 8, device="cuda"), torch.zeros(32, 8, device="cuda")
    (db,) = torch.autograd.grad(linear_act(x, w, b), b, gy.cuda())
    ref = gy.double().sum(0)
    assert ((db.cpu().double() - ref).abs() <= 4 * 2.0 ** -24 * ref).all(), db
    # the norm's weights: as exact as 32 bits in each workgroup and one rounding
    for rows, cols in ((2708, 128), (20000, 64)):
        g = torch.Generator().manual_seed(5)
        x, gy = torch.randn(rows, cols, generator=g), torch.randn(rows, cols, generator=g)
        wl = torch.ones(cols).cuda().requires_grad_(True)
        (dw,) = torch.autograd.grad(rms_norm(x.cuda(), wl), wl, gy.cuda())
        terms = gy.double() * x.double() * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        # errors of the terms (a handful of roundings each) and of the workgroups' sums of at most 16 rows side by side add up like a walk
        off = (dw.cpu().double() - terms.sum(0)).norm() / terms.sum(0).norm()
        assert off <= 4 * 2.0 ** -24, off


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(100, 40000, 24), (300, 6000, 200), (257, 9001, 130), (70, 131071, 9), (1500, 1024, 1024), (40, 5000, 48)])
def test_sums_of_8_bit_integers_are_exact(rows, k, n):
    # sums past 2^24 in every part of a cut reduction, and past it altogether: one rounding to fp32, at the end
    g = torch.Generator().manual_seed(6)
    q, w = (torch.randint(90, 128, (m, k), dtype=torch.int8, generator=g) for m in (rows, n))
    w[::3] *= -1
    got = linear_q8(q.cuda(), torch.ones(rows).cuda(), w.cuda(), torch.ones(n).cuda(), dtype=torch.float32)
    assert torch.equal(got.cpu(), (q.double() @ w.double().t()).float())


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["relu", "gelu", "silu", "leaky_relu"])
@pytest.mark.parametrize("n", [16, 33])
def test_gradients_where_an_argument_leaves_fp16(name, n):
    # z of +-90,000 and +-60,000, and what lies between: the activation's slope is 0 or 1 (0.2 where the rows leak) whatever z is rounded to
    x = torch.tensor([[300.0], [200.0], [-200.0], [-300.0], [1.0]]).half()
    w = torch.full((n, 1), 300.0).half()
    xl, wl = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y = linear_act(xl, wl, activation=name)
    low = 0.2 if name == "leaky_relu" else 0.0
    assert torch.equal(y[1].cpu().float(), torch.full((n,), 60000.0)) and ((y[3].cpu().float() + 0.0 - low * -90000.0).abs() <= 16).all()
    gy = torch.full((5, n), 2.0 ** -10)
    dx, dw = torch.autograd.grad(y, (xl, wl), gy.half().cuda())
    slope = torch.tensor([1.0, 1.0, low, low, 1.0]).half().double()[:, None]
    dz = (gy.double() * slope).half().double()
    within(dx, dz @ w.double(), allowance(torch.float16, dz @ w.double(), dz.abs() @ w.double().abs(), 2.0 ** -11 * (dz.abs() @ w.double().abs())), "dx")
    within(dw, dz.t() @ x.double(), allowance(torch.float16, dz.t() @ x.double(), dz.abs().t() @ x.double().abs(), 2.0 ** -11 * (dz.abs().t() @ x.double().abs())), "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["gelu", "silu"])
def test_slopes_far_out(dtype, name):
    z = torch.tensor([-3e38, -1e20, -1000.0, -129.0, -100.0, -30.0, -9.0, -1.0, 0.0, 1.0, 9.0, 30.0, 100.0, 129.0, 1000.0, 1e20, 3e38], dtype=torch.float64).to(dtype)
    x = z[:, None].cuda().requires_grad_(True)
    (dx,) = torch.autograd.grad(linear_act(x, torch.ones(1, 1, device="cuda", dtype=dtype), activation=name), x, torch.ones(len(z), 1, device="cuda", dtype=dtype))
    zd = z.double().requires_grad_(True)
    (ref,) = torch.autograd.grad(act(zd, name).sum(), zd)
    # one rounding of dz, one of dx, and the approximation's own 1e-6 (exponentials of up to 128 in 32 bits: 2^-17 of what is left there)
    assert ((dx[:, 0].double().cpu() - ref).abs() <= 2.02 * {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dtype] * ref.abs() + 1e-6).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-17, 1e-14, 1e-10, 1.0, 1e10, 1e14, 1e17])
def test_gradient_of_the_norm_of_large_and_small_rows(dtype, size):
    g = torch.Generator().manual_seed(7)
    x = (torch.randn(9, 300, generator=g).double() * size).to(dtype)
    gy = (torch.randn(9, 300, generator=g) + x.double().float() / size).to(dtype)       # with a part along the row, which the second term takes away
    xl = x.cuda().requires_grad_(True)
    (dx,) = torch.autograd.grad(rms_norm(xl, eps=0.0), xl, gy.cuda())
    xd = x.double().requires_grad_(True)
    (ref,) = torch.autograd.grad(xd * xd.square().mean(-1, keepdim=True).rsqrt(), xd, gy.double())
    s, hd, gd = xd.detach().square().mean(-1, keepdim=True).rsqrt(), xd.detach(), gy.double()
    parts = (s * gd).abs() + (hd * s).abs() * s * (gd * hd * s).abs().mean(-1, keepdim=True)
    unit = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}[dtype]
    assert ((dx.double().cpu() - ref).abs() <= 1.01 * unit * ref.abs() + 16 * 2.0 ** -24 * parts).all()


def every_operator():
    x, r, w = (torch.randn(s).cuda() for s in ((12, 8), (12, 8), (8, 8)))
    q, s = quantize_rows(w)
    return x, {"rms_norm": lambda v: rms_norm(v, residual=r)[0], "rms_norm_q8": lambda v: rms_norm_q8(v)[1], "quantize_rows": lambda v: quantize_rows(v)[1],
               "linear_act": lambda v: linear_act(v, w, activation="gelu"), "linear_act's weights": lambda v: linear_act(r, v, activation="gelu"),
               "linear_q8": lambda v: linear_q8(q, s, q, s, residual=v[:8], dtype=torch.float32), "orthogonalize": lambda v: orthogonalize(v)}


@pytest.mark.gpu
def test_calls_are_not_left_out_of_a_record():
    from torch.fx.experimental.proxy_tensor import make_fx
    x, calls = every_operator()
    for name, call in calls.items():
        ref = call(x)
        for record in (lambda: torch.jit.trace(call, (x,), check_trace=False), lambda: make_fx(call)(x), lambda: make_fx(call, tracing_mode="fake")(x)):
            with pytest.raises(_lib.FgnnError, match="not recorded"):
                record()
        # what only looks on is no record, and a compiler that does not know the call leaves it as it is
        with FlopCounterMode(display=False):
            assert torch.equal(call(x), ref)
        assert torch.equal(torch.compile(call, backend="eager")(x), ref), name


@pytest.mark.gpu
def test_transforms_that_would_drop_derivatives_are_refused():
    from torch.autograd import forward_ad
    x, calls = every_operator()
    for name, call in calls.items():
        with forward_ad.dual_level():
            with pytest.raises(_lib.FgnnError, match="forward mode"):
                call(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v).sum())(x)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(torch.stack([x, x]))


@pytest.mark.parametrize("flags", [["--optimizer", "muon"], ["--eight-bit", "int8"], ["--eight-bit", "e4m3", "--residual-blocks", "0"],
                                   ["--optimizer", "muon", "--residual-blocks", "2", "--num-layers", "0"]])
def test_flags_for_blocks_that_are_not_there(flags, capsys):
    from ae_mlsys_gnn_amd.train import train_gatconv
    with pytest.raises(SystemExit):
        train_gatconv.main(["--dataset", "cora"] + flags)
    assert "residual" in capsys.readouterr().err


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_of_16_bit_matrices(dtype, nesterov):
    g = torch.Generator().manual_seed(8)
    shapes = [(40, 64), (64, 40), (40, 64), (100, 7)]
    ws = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).cuda()) for s in shapes]
    ref = [w.detach().double().cpu() for w in ws]
    buf = [torch.zeros_like(w) for w in ref]
    opt = Muon(ws, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.01)
    a, b, c = 3.4445, -4.7750, 2.0315
    for step in range(6):
        for i, w in enumerate(ws):
            grad = torch.randn(shapes[i], generator=g).to(dtype)
            w.grad = grad.cuda()
            buf[i] = 0.9 * buf[i] + grad.double()
            u = grad.double() + 0.9 * buf[i] if nesterov else buf[i]
            u = u / (u.norm() + 1e-7)
            for _ in range(5):
                gram = u @ u.t()
                u = a * u + (b * gram + c * gram @ gram) @ u
            ref[i] = ref[i] * (1 - 0.1 * 0.01) - 0.1 * max(1.0, shapes[i][0] / shapes[i][1]) ** 0.5 * u
        opt.step()
        if step == 2:
            # another optimizer goes on from what this one wrote down
            saved = opt.state_dict()
            opt = Muon(ws, lr=0.5)
            opt.load_state_dict(saved)
    unit = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    for w, r in zip(ws, ref):
        assert all(v.dtype is torch.float32 for v in opt.state[w].values())
        # the 32-bit weights as those of fp32 matrices, and the parameter one rounding from them
        assert float((opt.state[w]["weights"].double().cpu() - r).norm()) <= 1e-4 * float(r.norm())
        assert ((w.detach().double() - opt.state[w]["weights"].double()).abs() <= unit * opt.state[w]["weights"].double().abs() + 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decay_of_16_bit_matrices_adds_up(dtype):
    w = torch.nn.Parameter(torch.randn(16, 24, generator=torch.Generator().manual_seed(9)).to(dtype).cuda())
    first = w.detach().double()
    w.grad = torch.zeros_like(w)
    opt = Muon([w], lr=0.02, weight_decay=0.01)             # 2e-4 a step, below half a step of either type
    for _ in range(400):
        opt.step()
    unit = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    want = first * (1 - 2e-4) ** 400
    assert ((w.detach().double() - want).abs() <= (unit + 400 * 2.0 ** -23) * want.abs()).all()
    # weights that something else has written are what the next step starts from
    with torch.no_grad():
        w[3:7].fill_(2.0)
    opt.step()
    want[3:7] = 2.0
    want = want * (1 - 2e-4)
    assert ((w.detach().double() - want).abs() <= (unit + 401 * 2.0 ** -23) * want.abs()).all()


def test_muon_refuses_other_types():
    with pytest.raises(_lib.FgnnError, match="float64"):
        Muon([torch.nn.Parameter(torch.randn(5, 4, dtype=torch.float64))])


def test_muon_refuses_what_is_no_matrix_in_later_groups_too():
    opt = Muon([torch.nn.Parameter(torch.randn(5, 4))])
    for bad in (torch.randn(5), torch.randn(2, 5, 4), torch.randn(5, 4, dtype=torch.float64)):
        with pytest.raises(_lib.FgnnError):
            opt.add_param_group({"params": [torch.nn.Parameter(bad)]})
    assert len(opt.param_groups) == 1
    # matrices without elements have nothing to learn
    for shape in ((0, 4), (4, 0)):
        w = torch.nn.Parameter(torch.empty(shape))
        w.grad = torch.empty(shape)
        Muon([w]).step()


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_eight_bit_blocks_follow_the_type_of_the_features(eight, dtype):
    torch.manual_seed(10)
    block = ResidualBlock(96, 200).cuda()
    served = block.quantized(eight)
    kept = {name: t.clone() for name, t in served.state_dict().items()}
    served = torch.nn.Sequential(served).to(dtype)
    for name, t in served[0].state_dict().items():
        same = name in ("w1", "w2", "w1_scale", "w2_scale")
        assert t.dtype is (kept[name].dtype if same else dtype) and t.is_cuda
        assert not same or torch.equal(t.float(), kept[name].float())
    x = torch.randn(40, 96).cuda().to(dtype)
    got, ref = served(x), block(x.float())
    assert got.dtype is dtype and float((got.float() - ref).norm()) <= 0.1 * float(ref.norm())
    # to other memory and back
    assert served.cpu()[0].w1.device.type == "cpu" and torch.equal(served.cuda()(x), got)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(5, 70, 33), (300, 128, 256), (300, 129, 257)])
def test_small_fp32_operands(rows, k, n):
    # the parts of an operand from 2^-110 on lie in the range that holds all of their bits; below, the last part's step of 2^-133 is what each may be off by
    g = torch.Generator().manual_seed(11)
    w = torch.randn(n, k, generator=g)
    for exponent, step in ((-109, 0.0), (-120, 2.0 ** -133), (-126, 2.0 ** -133)):
        x = torch.randn(rows, k, generator=g).sign() * (1 + torch.rand(rows, k, generator=g)) * 2.0 ** exponent
        for a, b in ((x, w), (w, x)):
            ref, terms = a.double() @ b.double().t(), a.double().abs() @ b.double().abs().t()
            off = step * (w.double().abs().sum(-1) if b is w else w.double().abs().sum(-1)[:, None])
            within(linear_act(a.cuda(), b.cuda()), ref, allowance(torch.float32, ref, terms, off), "2^%d" % exponent)
