"""Group norm with an activation over channels-last features, and its gradient, against float64."""
import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.operators import group_norm

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(UNIT)
ACTIVATIONS = [None, "relu", "gelu", "silu", "leaky_relu"]
# one point, one channel, groups of one channel and of all, odd widths, groups that no vector fits, few and many samples, samples of more than one chunk
SHAPES = [(1, 1, 1, 1), (3, 1, 40, 4), (2, 5, 7, 7), (4, 33, 64, 8), (2, 64, 86, 2), (13, 143, 602, 14), (1, 4096, 24, 3), (2, 9000, 48, 4), (70, 9, 33, 11), (500, 1, 128, 4),
          (3, 1024, 128, 8), (2, 2, 8200, 2), (1, 3, 20000, 1), (1, 20011, 9, 3), (2, 700, 512, 32)]


def reference(x, groups, w, b, eps, act, gy=None):
    """Values, gradients and the scales of their errors: what sums and differences in 32 bits are made of."""
    n, c = x.shape[0], x.shape[-1]
    v = x.double().reshape(n, -1, groups, c // groups)
    w = (torch.ones(c) if w is None else w).double().view(groups, -1)
    b = (torch.zeros(c) if b is None else b).double().view(groups, -1)
    mean = v.mean((1, 3), keepdim=True)
    rstd = ((v - mean).square().mean((1, 3), keepdim=True) + eps).rsqrt()
    u = (v - mean) * rstd
    z = (u * w + b).requires_grad_(True)
    f = {None: lambda t: t * 1, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, "leaky_relu": lambda t: torch.nn.functional.leaky_relu(t, 0.2)}
    y = f[act](z)
    # u is off by roundings of itself, of the mean (in standard deviations) and of the sums
    su = u.abs() + mean.abs() * rstd + 1
    sz = su * w.abs() + b.abs()
    out = {"y": (y.detach(), sz)}
    if gy is not None:
        g = gy.double().reshape(v.shape)
        d, = torch.autograd.grad(y, z, g)
        z = z.detach()
        # where z is 0 to its error, relu's slope may be either
        open_ = g.abs() * (z.abs() <= 16 * 2.0 ** -24 * sz) * (act in ("relu", "leaky_relu"))
        sd = g.abs() * (1 + sz) + open_ * 2.0 ** 20
        dw = d * w
        dx = rstd * (dw - dw.mean((1, 3), keepdim=True) - u * (dw * u).mean((1, 3), keepdim=True))
        sw = sd * w.abs()
        out["dx"] = (dx, rstd * (sw + sw.mean((1, 3), keepdim=True) + su * (sw * su).mean((1, 3), keepdim=True)))
        out["dw"] = ((d * u).sum((0, 1)), (sd * su).sum((0, 1)))
        out["db"] = (d.sum((0, 1)), sd.sum((0, 1)))
    return out


def within(got, ref, unit, what):
    want, scale = (t.reshape(got.shape) for t in ref)
    got = got.detach().double().cpu()
    tol = unit * want.abs() * 1.01 + 16 * 2.0 ** -24 * scale + (2.0 ** -25 if unit == 2.0 ** -11 else 0)       # (fp16's smallest step)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), "%s: %d of %d, worst %.3g" % (what, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol).max()))


def check(x, groups, w, b, gy, act, eps=1e-5, lay=lambda t: t):
    leaves = [lay(x.cuda()).requires_grad_(True)] + [None if t is None else t.cuda().requires_grad_(True) for t in (w, b)]
    y = group_norm(leaves[0], groups, leaves[1], leaves[2], eps=eps, activation=act)
    assert y.dtype is x.dtype and y.shape == x.shape
    wanted = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None], torch.autograd.grad(y, wanted, gy.cuda())))
    ref = reference(x, groups, w, b, eps, act, gy)
    within(y, ref["y"], UNIT[x.dtype], "y")
    for name, got in grads.items():
        within(got, ref[name], UNIT[got.dtype], name)
    with torch.no_grad():
        assert torch.equal(group_norm(leaves[0], groups, leaves[1], leaves[2], eps=eps, activation=act), y)


def inputs(shape, channels, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * torch.exp(0.5 * torch.randn(channels, generator=g)) + torch.randn(channels, generator=g)).to(dtype)
    w, b = (1 + 0.3 * torch.randn(channels, generator=g)).to(dtype), (0.3 * torch.randn(channels, generator=g)).to(dtype)
    return x, w, b, torch.randn(shape, generator=g).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(dtype, shape):
    batch, points, channels, groups = shape
    x, w, b, gy = inputs((batch, points, channels), channels, dtype, points + channels)
    check(x, groups, w, b, gy, ACTIVATIONS[(points + channels) % 5])


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("dtype", TYPES)
def test_activations(act, dtype):
    x, w, b, gy = inputs((3, 50, 60), 60, dtype, 1)
    check(x, 5, w, b, gy, act)
    check(x, 5, w.float(), None, gy, act)
    check(x, 5, None, b.float(), gy, act)
    check(x, 5, None, None, gy, act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    x, w, b, gy = inputs((2, 6, 10, 48), 48, dtype, 2)
    check(x, 4, w, b, gy, "silu")                                                   # more dimensions
    wide = torch.zeros(2, 60, 101, dtype=dtype).cuda()
    def cut(t):
        view = wide[:, :, 3:51]
        view.copy_(t.view(2, 60, 48))
        return view.detach()
    flat, g = x.view(2, 60, 48), gy.view(2, 60, 48)
    check(flat, 4, w, b, g, "relu", lay=cut)                                        # rows that start anywhere
    check(flat, 4, w, b, g, "relu", lay=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2).detach())      # channels first in memory
    check(flat[:, :, :].transpose(0, 1), 4, w, b, g.transpose(0, 1), None, lay=lambda t: t.detach())            # samples inside points
    check(flat[:1].expand(3, 60, 48), 4, w, b, g[:1].expand(3, 60, 48), "gelu", lay=lambda t: t[:1].expand(3, 60, 48).detach())
    check(flat[:, 0], 4, w, b, g[:, 0], "gelu")                                     # no points


@pytest.mark.gpu
def test_gradient_against_differences():
    x, w, b, gy = inputs((2, 7, 12), 12, torch.float32, 3)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, b)]
    group_norm(leaves[0], 3, leaves[1], leaves[2], activation="silu").backward(gy.cuda())

    def value(*t):
        return float((reference(t[0], 3, t[1], t[2], 1e-5, "silu")["y"][0].reshape(gy.shape) * gy.double()).sum())
    step = 1e-5
    for which, leaf in enumerate(leaves):
        for at in range(0, leaf.numel(), 5):
            ends = []
            for sign in (1, -1):
                moved = [t.double().clone() for t in (x, w, b)]
                moved[which].view(-1)[at] += sign * step
                ends.append(value(*moved))
            # second order in the step, float64 rounding of a value of order 10 over the step, and the gradient's own 2^-20
            assert abs(float(leaf.grad.view(-1)[at]) - (ends[0] - ends[1]) / (2 * step)) < 3e-5


@pytest.mark.gpu
def test_far_means_and_constant_groups():
    g = torch.Generator().manual_seed(4)
    # a mean of 4096 deviations: the features themselves are given to 2^-12 deviations, and what is formed of them is no worse
    x = 4096 + torch.randn(2, 3000, 16, generator=g)
    w, b = torch.ones(16), torch.zeros(16)
    check(x, 2, w, b, torch.randn(x.shape, generator=g), None)
    # channels that lie far from one another in a group
    x = torch.randn(2, 500, 16, generator=g) + 100 * torch.arange(16)
    check(x, 2, w, b, torch.randn(x.shape, generator=g), "silu")
    y = group_norm(torch.full((2, 100, 8), 3.0).cuda(), 2, eps=1e-5)
    assert (y == 0).all()
    x = torch.randn(3, 40, 8, generator=g).cuda()
    x[1, 7, 2] = float("nan")
    x[2, 3, 6] = float("inf")
    y = group_norm(x, 2)
    assert torch.isfinite(y[0]).all() and y[1, :, :4].isnan().all() and torch.isfinite(y[1, :, 4:]).all() and torch.isfinite(y[2, :, :4]).all()
    assert not torch.isfinite(y[2, :, 4:]).any()


@pytest.mark.gpu
def test_nothing_to_do():
    w = torch.ones(8).cuda().requires_grad_(True)
    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.empty(shape).cuda().requires_grad_(True)
        y = group_norm(x, 2, w, w)
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty(shape).cuda())
        assert y.shape == dx.shape == shape and (dw == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 700, 512, 32), (1, 20011, 9, 3), (40, 30, 64, 8)])
def test_streams_repetitions_and_graphs(shape):
    batch, points, channels, groups = shape
    x, w, b, gy = (t.cuda() for t in inputs((batch, points, channels), channels, torch.float32, 5))
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def work():
        y = group_norm(*leaves[:1], groups, *leaves[1:], activation="gelu")
        return (y.detach(),) + torch.autograd.grad(y, leaves, gy)
    first = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(first, other))
    # one array alone gives what all of them give
    for i, leaf in enumerate(leaves):
        rest = [t if j == i else t.detach() for j, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(group_norm(rest[0], groups, rest[1], rest[2], activation="gelu"), leaf, gy)[0], first[1 + i])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        eager = [t.clone() for t in work()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, eager)), i


def test_refusals():
    x, w = torch.randn(2, 4, 8), torch.randn(8)
    with pytest.raises(_lib.FgnnError, match="no CPU path"):
        group_norm(x, 2, w)
    with pytest.raises(_lib.FgnnError, match="activation"):
        group_norm(x, 2, w, activation="tanh")
    l, p = _lib.lib(), 256
    def call(batch=2, points=4, cols=8, groups=2, type=0, x=p, ld=8, wt=0, act=0, y=p, ws=1 << 20):
        return l.fgnn_group_norm(batch, points, cols, groups, type, x, ld, 32, p, wt, None, 0, 1e-5, act, 0.2, y, p, p, p, ws, None)
    assert call(groups=3) == -2 and call(groups=0) == -2 and call(ld=7) == -2 and call(type=3) == -2 and call(type=1, wt=2) == -2 and call(act=5) == -2 and call(batch=-1) == -2
    assert call(x=None) == -1 and call(y=None) == -1 and call(points=100000, ws=0) == -5
    assert l.fgnn_group_norm_backward(2, 4, 8, 2, 0, p, p, 8, 32, p, 0, None, 0, 0, 0.2, p, p, p, p, None, p, 0, None) == -5
    assert l.fgnn_group_norm_backward(2, 4, 8, 2, 0, None, p, 8, 32, p, 0, None, 0, 0, 0.2, p, p, p, p, None, p, 1 << 20, None) == -1


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, w = torch.randn(2, 4, 8).cuda(), torch.randn(8).cuda()
    for bad in (lambda: group_norm(x, 3), lambda: group_norm(x, 0), lambda: group_norm(x.double(), 2), lambda: group_norm(x, 2, w[:7]), lambda: group_norm(x, 2, w.half()),
                lambda: group_norm(x, 2, w, w.cpu()), lambda: group_norm(x[0, 0], 2), lambda: group_norm(x[:, :, :0], 1), lambda: group_norm(x, -2)):
        with pytest.raises(_lib.FgnnError):
            bad()
    y = group_norm(x.requires_grad_(True), 2)
    grad, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="second order"):
        grad.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("points", [2, 15, 17, 63, 65, 129, 257, 513, 1025, 2303, 2305, 4097, 8191, 8193, 9216, 9217])
def test_sizes_of_samples(dtype, points):
    """Samples that a wave, a workgroup of 256 or of 512 threads and none of them holds, and the sizes next to where one takes over from another."""
    for channels, groups in ((16, 2), (40, 8), (21, 7)):
        x, w, b, gy = inputs((2, points, channels), channels, dtype, points)
        check(x, groups, w, b, gy, ACTIVATIONS[points % 5])


@pytest.mark.gpu
@pytest.mark.parametrize("channels,groups", [(512, 1), (513, 1), (1030, 2), (24, 24), (6, 1), (602, 43)])
def test_widths_of_groups(channels, groups):
    for dtype in TYPES:
        for batch, points in ((300, 3), (3, 400)):
            x, w, b, gy = inputs((batch, points, channels), channels, dtype, channels)
            check(x, groups, w, b, gy, "silu")


@pytest.mark.gpu
def test_calls_at_the_same_time():
    sets = [(groups, [t.cuda() for t in inputs((batch, points, channels), channels, torch.float32, seed)])
            for seed, (batch, points, channels, groups) in enumerate([(3, 20000, 64, 8), (40, 300, 128, 4), (1, 1, 9000, 3)])]

    def work(groups, arrays):
        leaves = [t.detach().requires_grad_(True) for t in arrays[:3]]
        y = group_norm(leaves[0], groups, leaves[1], leaves[2], activation="gelu")
        return (y.detach(),) + torch.autograd.grad(y, leaves, arrays[3])
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
