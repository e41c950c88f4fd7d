"""Attention to keys and values of another length, and its gradients, against float64."""
import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.operators import cross_attention

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(UNIT)
# samples, queries, keys, heads, heads of keys, components: one of each; lengths either side of tiles; few and many queries; shared heads; odd and the widest components; many keys
# for few queries, and the other way round
SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 77, 8, 2, 64), (3, 5, 33, 4, 4, 40), (2, 63, 64, 2, 2, 64), (1, 65, 65, 3, 3, 80), (2, 130, 31, 6, 2, 37), (1, 200, 129, 2, 1, 128), (2, 33, 300, 5, 5, 96),
          (1, 64, 5000, 2, 2, 64), (1, 3000, 40, 2, 1, 32), (2, 17, 97, 3, 1, 256), (1, 150, 70, 2, 2, 200), (4, 2, 1000, 12, 3, 128), (1, 300, 260, 1, 1, 16), (1, 129, 1, 2, 2, 100),
          (1, 7, 4100, 1, 1, 130)]


def reference(q, k, v, lengths=None, mask=None, scale=None, g=None):
    """Values and bounds of their errors.  With u the type's unit (0 inside for fp32) and e a row's relative error of exp(S) in 32 bits, 16 roundings of 1 + |S| summed by magnitude:
    a softmax weight is off by u + 2 e of itself, delta = rowsum(G Y) by what Y is off, a gradient of a score by u of itself and by what delta is off."""
    unit = UNIT[q.dtype]
    inside = 0 if q.dtype is torch.float32 else unit
    b, nq, h, d = q.shape
    nk, share = k.shape[1], h // k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    qd, kd, vd = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(share, 1), v.double().transpose(1, 2).repeat_interleave(share, 1)
    seen = torch.ones(b, nk, dtype=torch.bool)
    if lengths is not None:
        seen &= torch.arange(nk) < lengths.view(b, 1)
    if mask is not None:
        seen &= mask
    hidden = ~seen.view(b, 1, nk, 1)
    kd, vd = kd.masked_fill(hidden, 0), vd.masked_fill(hidden, 0)
    score = (qd @ kd.transpose(2, 3) * scale).masked_fill(hidden.transpose(2, 3), -torch.inf)
    p = torch.softmax(score, -1).nan_to_num(0.0)
    e = 16 * 2.0 ** -24 * (1 + (scale * qd.abs() @ kd.abs().transpose(2, 3)).amax(-1, keepdim=True)) if nk else torch.zeros(b, h, nq, 1, dtype=torch.float64)
    y, sy = p @ vd, p @ vd.abs()
    ey = (inside + 2 * e) * sy

    def back(t):
        return t.transpose(1, 2)

    def heads(t):
        return t.view(b, h // share, share, nk, d).sum(2).transpose(1, 2)
    step = 2.0 ** -25 if q.dtype is torch.float16 else 0        # (fp16's smallest step)
    out = {"y": (back(y), back(ey + unit * y.abs()) + step)}
    if g is not None:
        gd = g.double().transpose(1, 2)
        dp, delta = gd @ vd.transpose(2, 3), (gd * y).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        edelta = (gd.abs() * (ey + inside * y.abs())).sum(-1, keepdim=True) + 2 * e * (gd.abs() * sy).sum(-1, keepdim=True)
        eds = inside * ds.abs() + p * (edelta + 2 * e * (gd.abs() @ vd.abs().transpose(2, 3) + (gd.abs() * sy).sum(-1, keepdim=True)))
        ep = p * (inside + 2 * e)
        for name, value, error, form in (("dq", ds @ kd * scale, eds @ kd.abs() * scale, back), ("dk", ds.transpose(2, 3) @ qd * scale, eds.transpose(2, 3) @ qd.abs() * scale, heads),
                                         ("dv", p.transpose(2, 3) @ gd, ep.transpose(2, 3) @ gd.abs(), heads)):
            value, error = form(value), form(error)
            out[name] = (value, error + unit * value.abs() + step)
    return out


def within(got, ref, what):
    got, (want, tol) = got.detach().double().cpu(), ref
    bad = ~((got - want).abs() <= 1.01 * tol + 2.0 ** -60)
    assert not bool(bad.any()), "%s: %d of %d, worst %.3g" % (what, int(bad.sum()), bad.numel(), float(((got - want).abs() / (tol + 2.0 ** -60)).max()))


def check(q, k, v, g, lengths=None, mask=None, scale=None, lay=lambda t: t):
    on = [lay(t.cuda()).detach().requires_grad_(True) for t in (q, k, v)]
    hide = dict(lengths=None if lengths is None else lengths.cuda(), mask=None if mask is None else mask.cuda(), scale=scale)
    y = cross_attention(*on, **hide)
    assert y.shape == q.shape and y.dtype is q.dtype
    grads = torch.autograd.grad(y, on, lay(g.cuda()))
    ref = reference(q, k, v, lengths, mask, scale, g)
    within(y, ref["y"], "y")
    for name, got in zip(("dq", "dk", "dv"), grads):
        within(got, ref[name], name)
    with torch.no_grad():
        assert torch.equal(cross_attention(*on, **hide), y)
    return y, grads


def inputs(shape, dtype, seed=0):
    b, nq, nk, h, hk, d = shape
    g = torch.Generator().manual_seed(seed + nq + nk + d)
    return [torch.randn(s, generator=g).to(dtype) for s in ((b, nq, h, d), (b, nk, hk, d), (b, nk, hk, d), (b, nq, h, d))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(dtype, shape):
    check(*inputs(shape, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(5, 70, 200, 4, 2, 64), (5, 3, 513, 2, 2, 40), (5, 257, 65, 3, 1, 128)])
def test_lengths_and_masks(dtype, shape):
    b, nq, nk = shape[:3]
    q, k, v, g = inputs(shape, dtype)
    lengths = torch.tensor([nk, 0, 1, 64, nk - 1])
    gen = torch.Generator().manual_seed(3)
    mask = torch.rand(b, nk, generator=gen) < 0.5
    mask[3] = False
    for hide in (dict(lengths=lengths), dict(lengths=lengths.int()), dict(mask=mask), dict(lengths=lengths, mask=mask)):
        y, (dq, dk, dv) = check(q, k, v, g, **hide)
        seen = (torch.arange(nk) < lengths.view(b, 1) if "lengths" in hide else torch.ones(b, nk, dtype=torch.bool)) & hide.get("mask", torch.ones((), dtype=torch.bool))
        none = ~seen.any(1)
        assert (y[none.cuda()] == 0).all() and (dq[none.cuda()] == 0).all()
        assert (dk[~seen.cuda()] == 0).all() and (dv[~seen.cuda()] == 0).all()
        # what is not seen may be anything
        bad = torch.where(seen.view(b, nk, 1, 1), k, torch.nan), torch.where(seen.view(b, nk, 1, 1), v, torch.inf)
        on = [t.cuda().requires_grad_(True) for t in (q, *bad)]
        again = cross_attention(*on, **{n: t.cuda() for n, t in hide.items()})
        assert torch.equal(again, y)
        assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(again, on, g.cuda()), (dq, dk, dv)))
    # lengths beyond either end are cut to it
    assert torch.equal(cross_attention(q.cuda(), k.cuda(), v.cuda(), lengths=torch.tensor([nk + 9, -3, 1, 64, 2 ** 40]).cuda()),
                       cross_attention(q.cuda(), k.cuda(), v.cuda(), lengths=torch.tensor([nk, 0, 1, 64, nk]).cuda()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 100, 90, 4, 2, 64), (2, 4, 700, 4, 1, 48), (2, 40, 50, 2, 2, 33)])
def test_layouts(dtype, shape):
    q, k, v, g = inputs(shape, dtype)
    plain, grads = check(q, k, v, g)
    for lay in (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),                           # heads before positions
                lambda t: torch.stack([t, t], 2)[:, :, 0],                                          # one half of a product's result
                lambda t: torch.cat([t.new_zeros(t.shape[:3] + (1,)), t, t], 3)[..., 1:1 + t.shape[3]],        # rows that start anywhere
                lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),                           # positions before samples
                lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)):                          # components apart
        y, other = check(q, k, v, g, lay=lay)
        assert torch.equal(y, plain) and all(torch.equal(a, c) for a, c in zip(other, grads))
    # one set of keys for all samples, one query for all positions, a gradient that is one number
    on = [q[:, :1].cuda().expand(q.shape), k[:1].cuda().expand(k.shape), v[:1].cuda().expand(v.shape)]
    same = [t.contiguous().requires_grad_(True) for t in on]
    on = [t.detach().requires_grad_(True) for t in on]
    one = torch.ones((), dtype=dtype).cuda().expand(q.shape)
    for a, c in zip(torch.autograd.grad(cross_attention(*on), on, one), torch.autograd.grad(cross_attention(*same), same, one.contiguous())):
        assert torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores_and_scales(dtype):
    q, k, v, g = inputs((2, 40, 150, 2, 2, 32), dtype)
    check(q, k, v, g, scale=3.0)
    check(q, k, v, g, scale=1e-4)
    # scores far below and above 0: weights are relative to a row's largest
    check(q * 0 + 8, k * 0 - 8 + (torch.arange(150) % 3).view(1, 150, 1, 1).to(dtype), v, g)
    check(q, k, v * 0 + 1, g * 0 + 1)
    y = cross_attention(q.cuda(), k.cuda(), torch.ones_like(v).cuda())
    assert ((y.double() - 1).abs() <= 2 * UNIT[dtype] + 2.0 ** -20).all()


@pytest.mark.gpu
def test_gradient_against_differences():
    q, k, v, g = inputs((1, 3, 5, 2, 1, 4), torch.float32)
    on = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    cross_attention(*on, mask=torch.tensor([[True, True, False, True, True]]).cuda()).backward(g.cuda())

    def value(*t):
        return float((reference(*t, mask=torch.tensor([[True, True, False, True, True]]))["y"][0] * g.double()).sum())
    UNIT[torch.float64] = 2.0 ** -53
    step = 1e-5
    for which, leaf in enumerate(on):
        for at in range(0, leaf.numel(), 3):
            ends = []
            for sign in (1, -1):
                moved = [t.double().clone() for t in (q, k, v)]
                moved[which].view(-1)[at] += sign * step
                ends.append(value(*moved))
            # second order in the step, float64 rounding of a value of order 10 over the step, and the gradient's own 2^-20
            assert abs(float(leaf.grad.view(-1)[at]) - (ends[0] - ends[1]) / (2 * step)) < 2e-5


@pytest.mark.gpu
def test_nothing_to_do_and_values_that_are_no_numbers():
    q, k, v, g = (t.cuda().requires_grad_(True) for t in inputs((2, 4, 6, 2, 1, 8), torch.float32))
    y = cross_attention(q, k[:, :0], v[:, :0])
    assert (y == 0).all() and all((t == 0).all() for t in torch.autograd.grad(y, (q, k, v), g))
    y = cross_attention(q[:, :0], k, v)
    assert y.shape == (2, 0, 2, 8) and all((t == 0).all() for t in torch.autograd.grad(y, (k, v), g[:, :0]))
    assert cross_attention(q[:0], k[:0], v[:0]).shape == (0, 4, 2, 8)
    # a query that is no number spoils its own row alone
    bad = q.detach().clone()
    bad[0, 1, 1, 3] = float("nan")
    y, fine = cross_attention(bad, k, v), cross_attention(q, k, v)
    assert y[0, 1, 1].isnan().all()
    y[0, 1, 1] = fine[0, 1, 1]
    assert torch.equal(y, fine)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((2, 100, 90, 4, 2, 64), torch.bfloat16), ((2, 3, 3000, 4, 1, 48), torch.float16), ((1, 64, 5000, 2, 2, 64), torch.float32)])
def test_streams_repetitions_and_graphs(shape, dtype):
    on = [t.cuda() for t in inputs(shape, dtype)]
    leaves, g = [t.requires_grad_(True) for t in on[:3]], on[3]
    lengths = torch.full((shape[0],), shape[2] - 3, dtype=torch.int32).cuda()

    def work():
        y = cross_attention(*leaves, lengths=lengths)
        return (y.detach(),) + torch.autograd.grad(y, leaves, g)
    first = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(first, other))
    for i, leaf in enumerate(leaves):
        rest = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(cross_attention(*rest, lengths=lengths), leaf, g)[0], first[1 + i])
    graphs, outs = [], []
    for _ in range(2):                      # two graphs, whose workspaces are their own
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(work())
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn_like(leaves[0]))
            lengths.fill_(shape[2] // (i + 1))
        eager = [t.clone() for t in work()]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for out in outs for a, c in zip(out, eager)), i


def test_refusals():
    q, k, v, _ = inputs((1, 2, 3, 2, 1, 8), torch.float32)
    with pytest.raises(_lib.FgnnError, match="no CPU path"):
        cross_attention(q, k, v)
    import ctypes
    l, p, st = _lib.lib(), 256, (ctypes.c_int64 * 12)(*([64, 16, 8] * 4))
    def forward(batch=1, nq=2, nk=3, heads=2, kv=1, dim=8, type=0, q=p, k=p, y=p, scale=1.0, strides=st, ws=None, n=0):
        return l.fgnn_attention(batch, nq, nk, heads, kv, dim, type, q, k, p, strides, None, 0, None, scale, y, None, ws, n, None)
    assert forward(kv=3) == -2 and forward(nq=-1) == -2 and forward(dim=0) == -2 and forward(type=3) == -2 and forward(scale=0.0) == -2 and forward(scale=float("nan")) == -2
    assert forward(dim=257) == -4 and forward(q=None) == -1 and forward(k=None) == -1 and forward(y=None) == -1 and forward(strides=None) == -1
    assert forward(dim=7) == -5                                                     # rows to be laid out anew, and no room
    def backward(dq=p, dk=p, dv=p, ws=p, n=1 << 20, lse=p):
        return l.fgnn_attention_backward(1, 2, 3, 2, 1, 8, 0, p, p, p, p, p, st, None, 0, None, 1.0, lse, dq, dk, dv, ws, n, None)
    assert backward(dv=None) == -1 and backward(lse=None) == -1 and backward(ws=None, n=0) == -5


@pytest.mark.gpu
def test_refusals_on_the_device():
    q, k, v, g = (t.cuda() for t in inputs((2, 4, 6, 2, 1, 8), torch.float32))
    n, m = torch.tensor([1, 2]).cuda(), torch.ones(2, 6, dtype=torch.bool).cuda()
    wide = torch.randn(1, 2, 1, 257).cuda()
    for bad in (lambda: cross_attention(q.half(), k, v), lambda: cross_attention(q.double(), k.double(), v.double()), lambda: cross_attention(q, k[:1], v[:1]), lambda: cross_attention(q, k, v[:, :5]),
                lambda: cross_attention(q[..., :7], k, v), lambda: cross_attention(q[0], k[0], v[0]), lambda: cross_attention(q, k.expand(2, 6, 3, 8), v.expand(2, 6, 3, 8)),
                lambda: cross_attention(q, k, v, lengths=n[:1]), lambda: cross_attention(q, k, v, lengths=n.float()), lambda: cross_attention(q, k, v, lengths=n.cpu()),
                lambda: cross_attention(q, k, v, mask=m[:, :5]), lambda: cross_attention(q, k, v, mask=m.int()), lambda: cross_attention(q, k, v, scale=0.0),
                lambda: cross_attention(q, k, v, scale=-1.0), lambda: cross_attention(q, k, v, scale=float("nan")), lambda: cross_attention(wide, wide, wide),
                lambda: cross_attention(q, k[:, :, :0], v[:, :, :0])):
        with pytest.raises(_lib.FgnnError):
            bad()
    q.requires_grad_(True)
    grad, = torch.autograd.grad(cross_attention(q, k, v).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="second order"):
        grad.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 31, 63, 65, 72, 127, 129, 136, 255])
def test_components_around_padded_widths(dtype, dim):
    check(*inputs((1, 37, 45, 4, 2, dim), dtype))
    check(*inputs((2, 2, 300, 2, 1, dim), dtype), lengths=torch.tensor([299, 130]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 3000, 4, 4, 128), (1, 20, 2500, 2, 1, 256), (1, 40, 900, 3, 3, 130), (2, 33, 1100, 2, 2, 64), (1, 65, 1500, 1, 1, 60), (2, 900, 33, 2, 1, 256)])
def test_few_rows_and_parts(dtype, shape):
    check(*inputs(shape, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rise", [0.0, 0.02, 0.3, -0.3])
def test_scores_that_rise_and_fall(dtype, rise):
    """A row's largest score moves on by less and by more than what sums are left unscaled for, in each of its tiles."""
    q, k, v, g = inputs((1, 70, 700, 2, 2, 40), dtype)
    q[..., 0], k[..., 0] = 1.0, (rise * torch.arange(700)).view(1, 700, 1).to(dtype)
    check(q, k, v, g, scale=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("power", [-12, 0, 6])
def test_small_and_large_gradients(dtype, power):
    q, k, v, g = inputs((2, 90, 1500, 2, 1, 64), dtype)
    check(q, k, v, (g.float() * 2.0 ** power).to(dtype))


@pytest.mark.gpu
def test_many_keys_of_many_samples_and_heads():
    b, nk, h, d = 32, 16384, 32, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(s, generator=g, device="cuda").bfloat16() for s in ((b, 1, h, d), (b, nk, h, d), (b, nk, h, d)))
    y = cross_attention(q, k, v).double()
    for i in (0, 13, 31):
        w = torch.softmax((q[i].double() * k[i].double()).sum(-1) * d ** -0.5, 0).unsqueeze(-1)
        want, size = (w * v[i].double()).sum(0), (w * v[i].double().abs()).sum(0)
        # weights rounded to the type, sums in 32 bits, the result rounded to the type
        assert ((y[i, 0] - want).abs() <= 1.01 * 2.0 ** -8 * (size + want.abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_offsets_past_32_bits(dtype):
    """Samples, and positions, that lie far apart in memory."""
    q, k, v, g = inputs((2, 40, 60, 2, 2, 64), dtype)
    far = torch.empty(2 ** 31 + 2 ** 20, dtype=dtype, device="cuda")

    def samples(t):
        out = far.as_strided(t.shape, (2 ** 31, *t.stride()[1:]), 64)
        return out.copy_(t)

    def positions(t):
        out = far.as_strided(t.shape, (64, 2 ** 25, t.stride(2) * 2, 1), 8)
        return out.copy_(t)
    plain = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    y = cross_attention(*plain)
    grads = torch.autograd.grad(y, plain, g.cuda())
    within(y, reference(q, k, v)["y"], "y")
    for lay in (samples, positions):
        for which in range(3):
            on = [t.detach() for t in plain]
            on[which] = lay(on[which]).detach()
            on = [t.requires_grad_(True) for t in on]
            again = cross_attention(*on)
            assert torch.equal(again, y)
            assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(again, on, g.cuda()), grads))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_calls_at_the_same_time(dtype):
    sets = [[t.cuda() for t in inputs(shape, dtype, seed)] for seed, shape in enumerate([(2, 300, 400, 4, 2, 64), (2, 5, 4000, 4, 2, 64), (1, 64, 3000, 2, 2, 96)])]

    def work(q, k, v, g):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        y = cross_attention(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, g)
    alone = [work(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    both = []
    for _ in range(3):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                both.append(work(*s))
    torch.cuda.synchronize()
    for i, got in enumerate(both):
        assert all(torch.equal(a, c) for a, c in zip(got, alone[i % len(sets)]))


@pytest.mark.gpu
def test_one_set_of_features_three_times():
    x = torch.randn(2, 70, 4, 32, generator=torch.Generator().manual_seed(1))
    leaf, g = x.cuda().requires_grad_(True), torch.randn(x.shape).cuda()
    apart = [x.cuda().requires_grad_(True) for _ in range(3)]
    once, = torch.autograd.grad(cross_attention(leaf, leaf, leaf), leaf, g)
    dq, dk, dv = torch.autograd.grad(cross_attention(*apart), apart, g)
    # three terms, added in one order or another
    assert ((once - (dq + dk + dv)).abs() <= 2.0 ** -22 * (dq.abs() + dk.abs() + dv.abs())).all()


@pytest.mark.gpu
def test_many_small_samples():
    b, h, d = 1 << 20, 16, 8
    q, k, v = (torch.randn(b, 1, h, d, device="cuda").bfloat16() for _ in range(3))
    assert torch.equal(cross_attention(q, k, v), v)             # one key's weight is 1
    with pytest.raises(RuntimeError, match="workgroups"):     # 2^24 of four waves: more threads than a launch has
        q.requires_grad_(True), v.requires_grad_(True)
        torch.autograd.grad(cross_attention(q, k, v), v, v.detach())


def test_strides_that_are_refused():
    import ctypes
    l, p, st = _lib.lib(), 256, (ctypes.c_int64 * 12)(*([64, 16, 8] * 4))
    st[4] = -16
    assert l.fgnn_attention(1, 2, 3, 2, 1, 8, 0, p, p, p, st, None, 0, None, 1.0, p, None, None, 0, None) == -2
    assert l.fgnn_attention_backward(1, 2, 3, 2, 1, 8, 0, p, p, p, p, p, st, None, 0, None, 1.0, p, p, p, p, p, 1 << 20, None) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 7, 33, 100, 131, 251])
def test_rows_at_the_end_of_their_memory(dtype, dim):
    """Rows of odd lengths, the last of which ends where its memory does, with queries and without any."""
    q, k, v, g = inputs((1, 3, 2, 1, 1, dim), dtype)
    check(q, k, v, g)
    on = [t.cuda().requires_grad_(True) for t in (q[:, :0], k, v)]
    y = cross_attention(*on)
    assert all((t == 0).all() for t in torch.autograd.grad(y, on[1:], g[:, :0].cuda()))
