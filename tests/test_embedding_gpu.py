"""Rows of a table by tokens and the table's gradient, against float64."""
import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.operators import embedding

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(UNIT)
# tokens, vocabulary, channels: one of each, rows shorter and longer than a workgroup's, odd widths, more tokens than rows and fewer, tokens that no row is met of
SHAPES = [(1, 1, 1), (1, 1000, 4096), (7, 3, 5), (300, 41, 128), (5000, 2, 24), (1000, 5000, 33), (4099, 300, 602), (64, 64, 8200), (20000, 1, 16), (33, 100, 1), (31, 5, 64), (70001, 513, 8)]


def gradient(tokens, vocabulary, gy, scale, padding=None):
    """The gradient and the sum of the magnitudes behind it."""
    t, g = tokens.reshape(-1).long(), gy.double().reshape(-1, gy.shape[-1])
    keep = (t >= 0) & (t < vocabulary)
    if padding is not None:
        keep &= t != padding
    out = torch.zeros(vocabulary, g.shape[1], dtype=torch.float64)
    return out.clone().index_add_(0, t[keep], g[keep] * scale), out.index_add_(0, t[keep], g[keep].abs() * abs(scale))


def within(got, want, unit, scale, what):
    got = got.detach().double().cpu()
    tol = unit * want.abs() * 1.01 + 2.0 ** -24 * scale + (2.0 ** -25 if unit == 2.0 ** -11 else 0)
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), "%s: %d of %d, worst %.3g" % (what, int(bad.sum()), bad.numel(), float(((got - want).abs() / tol).max()))


def check(tokens, w, gy, scale, padding=None):
    leaf = w.cuda().requires_grad_(True)
    y = embedding(tokens.cuda(), leaf, scale=scale, padding=padding)
    assert y.shape == tokens.shape + (w.shape[1],) and y.dtype is w.dtype
    want = w.double()[tokens.long()] * scale
    within(y, want, UNIT[w.dtype], 2 * want.abs(), "y")
    dw, = torch.autograd.grad(y, leaf, gy.cuda())
    want, sums = gradient(tokens, w.shape[0], gy, scale, padding)
    # a sum of n in 32 bits, in parts that are added up: its roundings are random, a handful of the sum of magnitudes at the most
    within(dw, want, UNIT[w.dtype], 16 * sums, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(dtype, shape):
    n, vocabulary, channels = shape
    g = torch.Generator().manual_seed(n + channels)
    w, gy = torch.randn(vocabulary, channels, generator=g).to(dtype), torch.randn(n, channels, generator=g).to(dtype)
    tokens = torch.randint(0, vocabulary, (n,), generator=g)
    check(tokens, w, gy, 1.0)
    check(tokens.int(), w, gy, channels ** 0.5, padding=int(tokens[0]))
    # a few tokens in most of the places, runs of every length
    skewed = (vocabulary * torch.rand(n, generator=g) ** 6).long()
    check(skewed, w, gy, -0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("runs", [[32] * 4, [31, 1, 32, 33, 64, 65, 1, 1], [200, 1, 200], [1, 31, 32, 96, 95], [16] * 20, [3000, 5000]])
def test_runs_that_end_at_and_inside_tiles(runs):
    tokens = torch.cat([torch.full((r,), 3 * i) for i, r in enumerate(runs)])
    g = torch.Generator().manual_seed(len(runs))
    w, gy = torch.randn(3 * len(runs) + 2, 20, generator=g), torch.randn(len(tokens), 20, generator=g)
    check(tokens, w, gy, 2.0)
    check(tokens, w, gy, 2.0, padding=3)
    check(tokens[torch.randperm(len(tokens), generator=g)], w, gy, 2.0, padding=0)


@pytest.mark.gpu
def test_shapes_strides_and_tokens_outside():
    g = torch.Generator().manual_seed(1)
    table = torch.randn(50, 70, generator=g)
    w = table[:, 3:40]
    tokens = torch.randint(0, 50, (4, 6), generator=g)
    gy = torch.randn(4, 6, 37, generator=g)
    check(tokens, w, gy, 1.5)
    check(tokens.t(), w, gy.transpose(0, 1), 1.5)
    leaf = w.cuda().requires_grad_(True)
    assert torch.equal(embedding(tokens.cuda(), table.cuda()[:, 3:40]), embedding(tokens.cuda(), leaf))
    one = torch.autograd.grad(embedding(tokens.cuda(), leaf), leaf, torch.ones(()).cuda().expand(4, 6, 37))[0]
    assert torch.equal(one, torch.autograd.grad(embedding(tokens.cuda(), leaf), leaf, torch.ones(4, 6, 37).cuda())[0])
    assert embedding(torch.tensor(7).cuda(), leaf).shape == (37,)
    bad = tokens.clone()
    bad[0, 0], bad[1, 1], bad[2, 2] = -1, 50, 2 ** 40
    y = embedding(bad.cuda(), leaf)
    outside = (bad < 0) | (bad >= 50)
    assert y[outside].isnan().all() and torch.equal(y[~outside], leaf[bad[~outside].cuda()])
    dw, = torch.autograd.grad(y, leaf, gy.cuda())
    want, sums = gradient(bad, 50, gy, 1.0)
    within(dw, want, UNIT[torch.float32], 16 * sums, "dw")


@pytest.mark.gpu
def test_nothing_to_do():
    w = torch.randn(5, 8).cuda().requires_grad_(True)
    y = embedding(torch.empty(0, 3, dtype=torch.int64).cuda(), w)
    dw, = torch.autograd.grad(y, w, torch.empty(0, 3, 8).cuda())
    assert y.shape == (0, 3, 8) and (dw == 0).all()
    none = torch.empty(0, 8).cuda().requires_grad_(True)
    y = embedding(torch.tensor([0, 1]).cuda(), none)
    assert y.isnan().all() and torch.autograd.grad(y, none, torch.ones(2, 8).cuda())[0].shape == (0, 8)


@pytest.mark.gpu
def test_streams_repetitions_and_graphs():
    tokens = (40 * torch.rand(30000) ** 3).long().cuda()
    w, gy = torch.randn(41, 64).cuda().requires_grad_(True), torch.randn(30000, 64).cuda()

    def work():
        y = embedding(tokens, w, scale=8.0, padding=3)
        return y.detach(), torch.autograd.grad(y, w, gy)[0]
    first = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(3):
        tokens.copy_((40 * torch.rand(30000) ** (i + 1)).long())
        eager = [t.clone() for t in work()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


def test_refusals():
    with pytest.raises(_lib.FgnnError, match="no CPU path"):
        embedding(torch.zeros(3, dtype=torch.int64), torch.randn(4, 8))
    l, p = _lib.lib(), 256
    assert l.fgnn_embedding(-1, 4, 8, 0, p, 1, p, 8, 1.0, p, None) == -2 and l.fgnn_embedding(2, 4, 8, 3, p, 1, p, 8, 1.0, p, None) == -2
    assert l.fgnn_embedding(2, 4, 8, 0, p, 1, p, 7, 1.0, p, None) == -2 and l.fgnn_embedding(2, 4, 8, 0, None, 1, p, 8, 1.0, p, None) == -1
    assert l.fgnn_embedding(2, 4, 8, 0, p, 1, p, 8, 1.0, None, None) == -1 and l.fgnn_embedding(1 << 31, 4, 8, 0, p, 1, p, 8, 1.0, p, None) == -4
    assert l.fgnn_embedding_backward(300, 4, 8, 0, p, 1, -1, p, 8, 1.0, p, None, 0, None) == -5
    assert l.fgnn_embedding_backward(2, 4, 8, 0, p, 1, -1, p, 7, 1.0, p, p, 1 << 20, None) == -2


@pytest.mark.gpu
def test_refusals_on_the_device():
    t, w = torch.zeros(3, dtype=torch.int64).cuda(), torch.randn(4, 8).cuda()
    for bad in (lambda: embedding(t.float(), w), lambda: embedding(t.short(), w), lambda: embedding(t, w.double()), lambda: embedding(t, w[0]), lambda: embedding(t.cpu(), w),
                lambda: embedding(t, w, padding=4), lambda: embedding(t, w, padding=-1), lambda: embedding(t, w[:, :0])):
        with pytest.raises(_lib.FgnnError):
            bad()
    w.requires_grad_(True)
    grad, = torch.autograd.grad(embedding(t, w).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="second order"):
        grad.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [2, 63, 255, 256, 257, 1023, 1025, 4095, 4096, 4097, 8193])
def test_numbers_of_tokens(dtype, n):
    """Either side of where another way of sorting takes over, with tokens that all are one, that all differ, and of int32's whole range."""
    g = torch.Generator().manual_seed(n)
    w, gy = torch.randn(n + 3, 9, generator=g).to(dtype), torch.randn(n, 9, generator=g).to(dtype)
    check(torch.full((n,), n + 2), w, gy, 1.0)
    check(torch.randperm(n + 3, generator=g)[:n], w, gy, 0.5, padding=1)
    wild = torch.randint(-2 ** 31, 2 ** 31 - 1, (n,), generator=g).int()
    wild[::3] = n
    leaf = w.cuda().requires_grad_(True)
    y = embedding(wild.cuda(), leaf)
    dw, = torch.autograd.grad(y, leaf, gy.cuda())
    want, sums = gradient(wild, n + 3, gy, 1.0)
    within(dw, want, UNIT[dtype], 16 * sums, "dw")
    assert y[(wild < 0) | (wild >= n + 3)].isnan().all()


@pytest.mark.gpu
def test_calls_at_the_same_time():
    g = torch.Generator().manual_seed(1)
    sets = [(torch.randint(0, rows, (n,), generator=g).cuda(), torch.randn(rows, 64, generator=g).cuda(), torch.randn(n, 64, generator=g).cuda()) for n, rows in ((30000, 41), (3000, 900), (9000, 20000))]

    def work(tokens, w, gy):
        leaf = w.detach().requires_grad_(True)
        return torch.autograd.grad(embedding(tokens, leaf), leaf, gy)[0]
    alone = [work(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    both = []
    for _ in range(3):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                both.append(work(*s))
    torch.cuda.synchronize()
    assert all(torch.equal(got, alone[i % len(sets)]) for i, got in enumerate(both))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_few_tokens_of_large_and_wide_tables(dtype):
    g = torch.Generator().manual_seed(2)
    for n, vocabulary, channels in ((200, 16384, 8), (256, 16385, 12), (256, 60000, 3), (256, 41000, 103), (256, 8192, 1024), (256, 8193, 1024), (250, 5, 5000), (256, 1, 70), (100, 40, 2050)):
        w, gy = torch.randn(vocabulary, channels, generator=g).to(dtype), torch.randn(n, channels, generator=g).to(dtype)
        tokens = torch.randint(0, vocabulary, (n,), generator=g)
        tokens[:3] = torch.tensor([0, vocabulary - 1, vocabulary - 1])
        check(tokens, w, gy, 0.7)
        check(tokens.int(), w, gy, 0.7, padding=0)
