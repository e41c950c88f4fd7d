"""The conditioned blocks' operators where sizes, values and calls are out of the ordinary."""
import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.operators import cross_attention, embedding, group_norm
from . import test_attention_gpu as attention, test_group_norm_gpu as norm


@pytest.mark.gpu
@pytest.mark.parametrize("channels,dtype", [(261121, torch.float32), (262146, torch.float32), (522241, torch.bfloat16), (522247, torch.float16)])
@pytest.mark.parametrize("points", [1, 2])
def test_rows_whose_last_part_is_less_than_a_vector(channels, dtype, points):
    """Rows that workgroups share, with one to seven channels left for the last of them."""
    x, w, b, gy = norm.inputs((2, points, channels), channels, dtype, points)
    norm.check(x, 1, w, b, gy, "silu")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 20000, 16, 2), (1, 70000, 8, 1), (2, 700, 1200, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_points_far_from_the_others(dtype, shape):
    """A point that lies far out, in all channels or in one, as the first and in the middle, and features far from 0 behind a first point of zeros, in samples that go in parts."""
    batch, points, channels, groups = shape
    x, w, b, gy = norm.inputs((batch, points, channels), channels, dtype, 7)
    for at in (0, points // 2):
        for size in (100.0, 1000.0, 1e4):
            for where in (slice(None), 3):
                far = x.clone()
                far[:, at, where] = size
                norm.check(far, groups, w, b, gy, "silu")
    for mean in (100.0, 1000.0):
        far = (x.float() + mean).to(dtype)
        far[:, 0] = 0
        norm.check(far, groups, w, b, gy, None)


def test_workspaces_of_sizes_that_are_refused():
    """A caller asks for the workspace before the call that refuses the sizes."""
    import ctypes
    l, s, most = _lib.lib(), (ctypes.c_int64 * 12)(*([64, 16, 8] * 4)), 2 ** 31 - 1
    for cols, groups in ((4, 8), (10, 4), (8, 0), (0, 1), (most, 1), (most, most), (2 ** 30 + 1, 1)):
        assert l.fgnn_group_norm_workspace_bytes(2, 100000, cols, groups, 0) == 0 and l.fgnn_group_norm_backward_workspace_bytes(2, 100000, cols, groups, 0) == 0
        assert l.fgnn_group_norm(2, 100000, cols, groups, 0, 256, cols, cols, None, 0, None, 0, 1e-5, 0, 0.2, 256, 256, 256, None, 0, None) in (-2, -4)
    for n, vocabulary, cols in ((1000, 7, most), (1000, 7, 2 ** 30 + 1), (2 ** 40, 7, 8), (1000, 2 ** 30, 8), (1000, 7, 0)):
        assert l.fgnn_embedding_backward_workspace_bytes(n, vocabulary, cols, 0) == 0
        assert l.fgnn_embedding_backward(n, vocabulary, cols, 0, 256, 1, -1, 256, max(cols, 1), 1.0, 256, None, 0, None) in (-2, -4)
    for nq, nk, heads, kv in ((most, 5, 1, 1), (5, most, 1, 1), (2 ** 30, 5, 2, 1), (5, 5, 3, 2), (5, 5, 1, 0)):
        assert l.fgnn_attention_workspace_bytes(1, nq, nk, heads, kv, 8, 0, 256, 256, s) == 0
        assert l.fgnn_attention_backward_workspace_bytes(1, nq, nk, heads, kv, 8, 0, 256, 256, 256, 256, s) == 0
        assert l.fgnn_attention(1, nq, nk, heads, kv, 8, 0, 256, 256, 256, s, None, 0, None, 1.0, 256, None, None, 0, None) in (-2, -4)


def test_the_backward_pass_says_ahead_what_it_refuses():
    check, few, many = _lib.lib().fgnn_attention_backward_check, (2 ** 20 - 1, 1, 128, 16, 16, 8, 1), (2 ** 20, 1, 1, 16, 16, 8, 1)
    assert check(*few, 1, 1) == 0 and check(*many, 1, 0) == 0 and check(*many, 0, 0) == 0
    assert check(*many, 0, 1) == -4 and check(2 ** 19, 1, 129, 16, 16, 8, 1, 1, 1) == -4
    assert check(2 ** 20, 1, 0, 16, 16, 8, 1, 1, 1) == 0 and check(0, 1, 1, 16, 16, 8, 1, 1, 1) == 0        # nothing to launch
    assert check(1, 1, 1, 3, 2, 8, 1, 1, 1) == -2 and check(1, 1, 1, 1, 1, 257, 1, 1, 1) == -4


@pytest.mark.gpu
def test_calls_whose_gradients_are_refused_are_refused_before_they_run():
    b, h, d = 2 ** 20, 16, 8
    q, k, v = (torch.randn(b, 1, h, d, device="cuda").bfloat16() for _ in range(3))
    for leaf in (k, v):
        leaf.requires_grad_(True)
        with pytest.raises(_lib.FgnnError, match="workgroups"):
            cross_attention(q, k, v)
        with torch.no_grad():
            assert torch.equal(cross_attention(q, k, v), v)
        leaf.requires_grad_(False)
    # queries alone can be trained: the only key's weight is 1 whatever they are, so that the gradient is what two sums of eight products differ by, times a key
    q.requires_grad_(True)
    y = cross_attention(q, k, v)
    dq, = torch.autograd.grad(y, q, v)
    bound = 16 * 2.0 ** -24 * (v.float() * v.float()).sum(-1, keepdim=True) * k.float().abs() * d ** -0.5
    assert torch.equal(y.detach(), v) and (dq.float().abs() <= 1.01 * bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 256, 64, 2, 2, 64), (1, 256, 1024, 4, 2, 64), (1, 20, 4096, 4, 2, 128), (2, 200, 700, 2, 1, 36), (1, 100, 300, 1, 1, 256)])
@pytest.mark.parametrize("offset", [0.0, 4.0, -30.0])
def test_gradients_where_values_share_an_offset(dtype, shape, offset):
    """rowsum(G Y) is as large as the offset, and cancels against dP.  Bounds in the norm: a rounding to the type, of relative size u at most, is u / 3^1/2 in the mean square at most.
    There is one of every softmax weight in Y (of which delta is formed: delta is off by the sum over keys of P (G V) times it, a number a row), of every dS, and of the result."""
    b, nq, nk, h, hk, d = shape
    q, k, v, g = attention.inputs(shape, dtype)
    v = (v.float() + offset).to(dtype)
    on = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(cross_attention(*on), on[:2], g.cuda())
    share, scale, unit = h // hk, d ** -0.5, attention.UNIT[dtype] ** 2 / 3
    q, g = (t.double().transpose(1, 2) for t in (q, g))
    k, v = (t.double().transpose(1, 2).repeat_interleave(share, 1) for t in (k, v))
    p, dp = torch.softmax(q @ k.transpose(2, 3) * scale, -1), g @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    delta = unit * (p * dp).square().sum(-1, keepdim=True)

    def heads(t):
        return t.view(b, hk, share, nk, d).sum(2)
    dq, dk = ds @ k * scale, heads(ds.transpose(2, 3) @ q * scale)
    square_q = scale ** 2 * (unit * ds.square() @ k.square() + delta * (p @ k).square()) + unit * dq.square()
    square_k = heads(scale ** 2 * (unit * ds.square().transpose(2, 3) @ q.square() + p.square().transpose(2, 3) @ (delta * q.square()))) + unit * dk.square()
    for name, a, want, square in (("dq", got[0], dq, square_q), ("dk", got[1], dk, square_k)):
        off = float((a.double().cpu().transpose(1, 2) - want).norm())
        assert off <= float(square.sum().sqrt()), "%s: off by %.3g of its norm, %.2f of the bound" % (name, off / float(want.norm()), off / float(square.sum().sqrt()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)])
def test_attention_entries_that_keep_no_rest(dtype, code):
    """The C entries without it: the same values, gradients of values and (fp32) of all, and those of queries and keys within the bound for a rounded y."""
    import ctypes
    shape = (2, 70, 130, 4, 2, 64)
    b, nq, nk, h, hk, d = shape
    q, k, v, g = attention.inputs(shape, dtype)
    on = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    want_y = cross_attention(*on)
    want = torch.autograd.grad(want_y, on, g.cuda())
    l, gd = _lib.lib(), g.cuda()
    strides = (ctypes.c_int64 * 12)(*[s for t in (*on, gd) for s in t.stride()[:3]])
    y, lse, grads = torch.empty_like(want_y), torch.empty(b, h, nq, device="cuda"), [torch.empty_like(t) for t in on]
    sizes, p, stream = (b, nq, nk, h, hk, d, code), [t.data_ptr() for t in on], torch.cuda.current_stream().cuda_stream
    n = l.fgnn_attention_workspace_bytes(*sizes, p[1], p[2], strides)
    space = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    assert l.fgnn_attention(*sizes, *p, strides, None, 0, None, d ** -0.5, y.data_ptr(), lse.data_ptr(), space.data_ptr(), n, stream) == 0
    assert torch.equal(y, want_y)
    n = l.fgnn_attention_backward_workspace_bytes(*sizes, *p, gd.data_ptr(), strides)
    space = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    assert l.fgnn_attention_backward(*sizes, *p, y.data_ptr(), gd.data_ptr(), strides, None, 0, None, d ** -0.5, lse.data_ptr(), *[t.data_ptr() for t in grads], space.data_ptr(), n,
                                     stream) == 0
    assert torch.equal(grads[2], want[2])
    ref = attention.reference(q, k, v, g=g)
    for name, got, same in zip(("dq", "dk"), grads, want):
        attention.within(got, ref[name], name)
        assert torch.equal(got, same) == (dtype is torch.float32)


def every_operator():
    """Calls of one set of features each, by the operand that it is."""
    x, w, other = (torch.randn(s).cuda() for s in ((12, 4, 8), (8,), (12, 4, 8)))
    tokens, heads = torch.tensor([3, 0, 3, 11]).cuda(), other.view(12, 4, 2, 4)
    n, m = torch.full((12,), 3).cuda(), torch.rand(12, 4).cuda() < 0.7
    return x, {"group_norm": lambda t: group_norm(t, 2, w, w, activation="silu"), "group_norm's weights": lambda t: group_norm(other, 2, t[0, 0], activation="gelu"),
               "group_norm's bias": lambda t: group_norm(other, 2, w, t[0, 0]), "embedding": lambda t: embedding(tokens, t.view(12, 32), scale=2.0, padding=3),
               "queries": lambda t: cross_attention(t.view(12, 4, 2, 4), heads, heads, lengths=n), "keys": lambda t: cross_attention(heads, t.view(12, 4, 2, 4), heads, mask=m),
               "values": lambda t: cross_attention(heads, heads, t.view(12, 4, 2, 4))}


@pytest.mark.gpu
def test_calls_are_not_left_out_of_a_record():
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    x, calls = every_operator()
    for name, call in calls.items():
        ref = call(x)
        for record in (lambda: torch.jit.trace(call, (x,), check_trace=False), lambda: make_fx(call)(x), lambda: make_fx(call, tracing_mode="fake")(x)):
            with pytest.raises(_lib.FgnnError, match="not recorded"):
                record()

        class Module(torch.nn.Module):
            def forward(self, t):
                return call(t)
        with pytest.raises(Exception):
            torch.export.export(Module(), (x,))
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
        # and gradients of second order say that they are not recorded
        leaf = x.clone().requires_grad_(True)
        first, = torch.autograd.grad(call(leaf).sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="second order"):
            first.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", attention.TYPES)
def test_long_samples_with_values_that_are_no_numbers(dtype):
    """They spoil their own sample's group alone, wherever they lie in it."""
    x = torch.randn(7, 20003, 16, generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
    fine = group_norm(x, 2, activation="silu")
    for value in (float("nan"), float("inf"), -float("inf")):
        bad = x.clone()
        spoilt = torch.zeros(7, 16, dtype=torch.bool, device="cuda")
        for sample, at in enumerate((0, 3, 9999, 20001, 20002)):
            bad[sample, at, 5 + sample] = value
            group = (5 + sample) // 8
            spoilt[sample, 8 * group:8 * group + 8] = True
        z = group_norm(bad, 2)
        assert not torch.isfinite(z.transpose(1, 2)[spoilt]).any()
        y = group_norm(bad, 2, activation="silu")
        assert torch.equal(y.transpose(1, 2)[~spoilt], fine.transpose(1, 2)[~spoilt])


@pytest.mark.gpu
@pytest.mark.parametrize("value", [0.0, 0.1, -3.0, 1e15])
@pytest.mark.parametrize("points", [9217, 50000, 300007])
def test_long_samples_that_are_constant(value, points):
    """Their mean is the value itself, and their variance 0."""
    x = torch.full((1, points, 8), value, device="cuda")
    y, mean, rstd = torch.empty_like(x), torch.empty(1, 2, device="cuda"), torch.empty(1, 2, device="cuda")
    l = _lib.lib()
    n = l.fgnn_group_norm_workspace_bytes(1, points, 8, 2, 0)
    space = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert n > 0 and l.fgnn_group_norm(1, points, 8, 2, 0, x.data_ptr(), 8, points * 8, None, 0, None, 0, 0.25, 0, 0.2, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), space.data_ptr(), n,
                                       torch.cuda.current_stream().cuda_stream) == 0
    assert (mean == torch.tensor(value)).all() and (rstd == 2).all()
    # a x + (b - mean a): one rounding of mean a
    assert (y.abs() <= 2.0 ** -24 * 2 * abs(value)).all()
