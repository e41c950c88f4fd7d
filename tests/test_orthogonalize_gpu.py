"""Orthogonalised updates against the iteration in float64."""
import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.operators import orthogonalize

USUAL = (3.4445, -4.7750, 2.0315)
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def reference(g, steps, coefficients, eps=1e-7):
    """The iteration in float64, and how far 22 significant bits may take the result (Frobenius norm): a step rounds X, A, B and their products, each to
    2^-22 of terms that are (a + |b| + |c|) |X| altogether, and later steps multiply what is off by no more than their slope at 0 or its largest."""
    x = g.double() / (g.double().norm() + eps)
    off = 2.0 ** -22 * float(x.norm())
    for i in range(steps):
        a, b, c = coefficients[i] if isinstance(coefficients[0], tuple) else coefficients
        gram = x @ x.t()
        slope = max(abs(a), abs(a + 3 * b + 5 * c), 1.0)
        off = off * slope + 2.0 ** -22 * (abs(a) + abs(b) + abs(c)) * float(x.norm())
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x, off


def compare(g, steps=5, coefficients=USUAL):
    got = orthogonalize(g.cuda(), steps=steps, coefficients=coefficients)
    assert got.shape == g.shape and got.dtype == g.dtype
    flat, out = g.reshape(-1, *g.shape[-2:]), got.cpu().reshape(-1, *g.shape[-2:]).double()
    for i in range(flat.shape[0]):
        ref, off = reference(flat[i], steps, coefficients)
        allowed = off + UNIT[g.dtype] * float(ref.norm()) + (2.0 ** -25 * ref.numel() ** 0.5 if g.dtype is torch.float16 else 0)
        assert float((out[i] - ref).norm()) <= allowed, "matrix %d: off by %.3g, %.3g allowed" % (i, float((out[i] - ref).norm()), allowed)
    return got


# either side of chunks, slabs and tiles, both orientations, vectors
SHAPES = [(1, 1), (1, 9), (9, 1), (7, 5), (8, 16), (16, 64), (33, 100), (100, 33), (64, 64), (65, 130), (130, 65), (128, 256), (256, 128), (129, 129), (41, 602), (602, 41),
          (300, 500), (520, 264), (17, 4000), (4000, 17)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(dtype, shape):
    g = torch.Generator().manual_seed(shape[0] * 31 + shape[1])
    compare(torch.randn(shape, generator=g).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 64, 128), (5, 100, 30), (2, 2, 40, 40), (12, 16, 16), (2, 300, 700)])
def test_batches(shape):
    g = torch.Generator().manual_seed(3)
    m = torch.randn(shape, generator=g) * torch.rand(shape[:-2] + (1, 1), generator=g)
    got = compare(m)
    alone = torch.stack([orthogonalize(v.cuda()) for v in m.reshape(-1, *shape[-2:])]).reshape(shape)
    assert torch.equal(got, alone)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1024, 1024), (700, 2100), (2100, 700)])
def test_larger_matrices(shape):
    g = torch.Generator().manual_seed(4)
    low = torch.randn(shape[0], 20, generator=g) @ torch.randn(20, shape[1], generator=g)
    got = compare(low + 0.5 * torch.randn(shape, generator=g))
    s = torch.linalg.svdvals(got.double().cpu())
    assert float(s.max()) < 1.3 and float(s.median()) > 0.6


@pytest.mark.gpu
def test_scales_steps_and_coefficients():
    g = torch.Generator().manual_seed(6)
    m = torch.randn(48, 80, generator=g)
    ref = orthogonalize(m.cuda())
    # a power of two moves no rounding but that of eps
    for k in (2.0 ** -20, 2.0 ** 30):
        assert float((orthogonalize((m * k).cuda(), eps=0.0) - orthogonalize(m.cuda(), eps=0.0)).norm()) == 0.0
    for steps in (1, 2, 7):
        compare(m, steps=steps)
    compare(m, steps=12, coefficients=(1.5, -0.5, 0.0))
    compare(m, steps=8, coefficients=(2.0, -1.5, 0.5))
    compare(m, steps=3, coefficients=((3.0, -3.2, 1.2), (2.5, -2.0, 0.6), (1.875, -1.25, 0.375)))
    # columns and rows in memory the other way, and a view
    assert torch.equal(orthogonalize(m.t().contiguous().cuda().t()), ref)
    wide = torch.randn(48, 100, generator=g).cuda()
    wide[:, 7:87] = m.cuda()
    assert torch.equal(orthogonalize(wide[:, 7:87]), ref)


@pytest.mark.gpu
def test_zeros_rank_one_and_values_that_are_no_numbers():
    assert (orthogonalize(torch.zeros(20, 30).cuda()) == 0).all()
    g = torch.Generator().manual_seed(7)
    u, v = torch.randn(50, 1, generator=g), torch.randn(1, 70, generator=g)
    compare(u @ v)
    bad = torch.randn(3, 20, 30, generator=g)
    bad[1, 4, 5] = float("nan")
    got = orthogonalize(bad.cuda())
    assert got[1].isnan().all() and torch.equal(got[[0, 2]], orthogonalize(bad[[0, 2]].cuda()))
    for shape in ((0, 5), (5, 0), (0, 4, 4)):
        assert orthogonalize(torch.empty(shape).cuda()).shape == shape


@pytest.mark.gpu
def test_other_streams():
    m = torch.randn(200, 300).cuda()
    ref = orthogonalize(m)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = orthogonalize(m)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)


def test_refusals():
    with pytest.raises(_lib.FgnnError):
        orthogonalize(torch.randn(4, 4))
    import ctypes
    l, p = _lib.lib(), 256
    c = (ctypes.c_float * 3)(*USUAL)
    need = l.fgnn_orthogonalize_workspace_bytes(2, 40, 50)
    assert need > 0 and l.fgnn_orthogonalize_workspace_bytes(0, 40, 50) == 0
    assert l.fgnn_orthogonalize(2, 40, 50, 0, p, 0, c, 1e-7, p, p, need, None) == -2
    assert l.fgnn_orthogonalize(2, 40, 50, 3, p, 1, c, 1e-7, p, p, need, None) == -2
    assert l.fgnn_orthogonalize(2, 40, 50, 0, None, 1, c, 1e-7, p, p, need, None) == -1
    assert l.fgnn_orthogonalize(2, 40, 50, 0, p, 1, c, 1e-7, p, p, need - 1, None) == -5
    assert l.fgnn_orthogonalize(65536, 4, 4, 0, p, 1, c, 1e-7, p, p, 1 << 40, None) == -4
    away = (ctypes.c_float * 9)(*((30.0, 1.0, 1.0) * 3))
    assert l.fgnn_orthogonalize(2, 40, 50, 0, p, 3, away, 1e-7, p, p, need, None) == -4


@pytest.mark.gpu
def test_refusals_on_the_device():
    m = torch.randn(4, 4).cuda()
    for bad in (lambda: orthogonalize(m.double()), lambda: orthogonalize(m[0]), lambda: orthogonalize(m, steps=0), lambda: orthogonalize(m, coefficients=(1.0, 2.0)),
                lambda: orthogonalize(m, steps=2, coefficients=(USUAL,)), lambda: orthogonalize(m, coefficients=()), lambda: orthogonalize(m, coefficients=(40.0, 3.0, 2.0))):
        with pytest.raises(_lib.FgnnError):
            bad()
