"""The largest tiles of the dense operators' products, with remainders on every side: every element against float64, on the device."""
import pytest
import torch

from ae_mlsys_gnn_amd.operators import linear_act, linear_q8, orthogonalize, quantize_rows

from .test_linear_gpu import UNIT, act, allowance
from .test_orthogonalize_gpu import USUAL, reference

# 17 x 17 tiles of 256 and more: one a compute unit at the least.  Rows of whole 16 bytes, which are moved as they lie, and odd ones, which are laid out anew
SIZES = [(4104, 4200, 4296), (4101, 4203, 4299)]


def within(got, ref, tol, what):
    off = (got.detach().double() - ref).abs() / tol
    assert bool((off <= 1).all()), "%s: %d of %d outside, worst %.3g of the allowance" % (what, int((~(off <= 1)).sum()), off.numel(), float(off.max()))


def product(a, b):
    return a @ b.contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("name", [None, "silu"])
def test_linear_maps_and_gradients(dtype, size, name):
    rows, k, n = size
    g = torch.Generator(device="cuda").manual_seed(rows)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device="cuda").normal_(0, std, generator=g).to(dtype)
    x, w, b, r, gy = normal(rows, k), normal(n, k, std=k ** -0.5), normal(n), normal(rows, n), normal(rows, n)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = linear_act(*leaves[:3], residual=leaves[3], activation=name)
    grads = torch.autograd.grad(y, leaves, gy)
    xd, wd, bd, rd, gd = (t.double() for t in (x, w, b, r, gy))
    z = (product(xd, wd.t()) + bd).requires_grad_(True)
    a = act(z, name)
    magnitude = product(xd.abs(), wd.abs().t()) + bd.abs() + rd.abs()
    ref = a.detach() + rd
    within(y, ref, allowance(dtype, ref, 2 * magnitude + z.detach().abs()), "y")
    dz = torch.autograd.grad(a, z, gd)[0] if name else gd
    # dz is formed from z in the rows' type and rounded to it (without an activation it is the gradient itself)
    off = 1.01 * UNIT[dtype] * dz.abs() + gd.abs() * (0.8 * UNIT[dtype] * z.detach().abs() + 16 * 2.0 ** -24 * (2 + magnitude)) if name else torch.zeros_like(dz)
    dx, dw, db = product(dz, wd), product(dz.t().contiguous(), xd), dz.sum(0)
    within(grads[0], dx, allowance(dtype, dx, product(dz.abs(), wd.abs()), product(off, wd.abs())), "dx")
    within(grads[1], dw, allowance(dtype, dw, product(dz.abs().t().contiguous(), xd.abs()), product(off.t().contiguous(), xd.abs())), "dw")
    within(grads[2], db, allowance(dtype, db, dz.abs().sum(0), off.sum(0)), "db")
    assert torch.equal(grads[3], gy)


@pytest.mark.gpu
@pytest.mark.parametrize("eight", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("size", SIZES + [(4101, 4208, 4299)])
def test_eight_bits(eight, size):
    rows, k, n = size
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, w, b, r = (torch.empty(s, device="cuda").normal_(generator=g) for s in ((rows, k), (n, k), (n,), (rows, n)))
    q, s = quantize_rows(x, eight)
    wq, ws = quantize_rows(w * k ** -0.5, eight)
    xd, wd = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None]
    z, magnitude = product(xd, wd.t()), product(xd.abs(), wd.abs().t()) + b.double().abs() + r.double().abs()
    for dtype, name, residual in ((torch.bfloat16, "gelu", r.bfloat16()), (torch.float16, None, None), (torch.float32, "relu", r)):
        y = linear_q8(q, s, wq, ws, b, residual=residual, activation=name, dtype=dtype)
        ref = act(z + b.double(), name) + (0 if residual is None else residual.double())
        within(y, ref, allowance(dtype, ref, 2 * magnitude + (z + b.double()).abs()), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2049, 4100), (4100, 2049), (2, 2049, 4100), (2, 4100, 2049), (6, 1100, 2300), (2304, 2304)])
def test_orthogonalised_updates(shape):
    # symmetric products on tiles of 256 whose reduction is cut, products by X on such tiles whole (batches) and smaller ones
    g = torch.Generator(device="cuda").manual_seed(shape[-1])
    m = torch.empty(shape, device="cuda").normal_(generator=g)
    m = m + 3 * torch.empty(shape[:-1] + (20,), device="cuda").normal_(generator=g) @ torch.empty(shape[:-2] + (20, shape[-1]), device="cuda").normal_(generator=g)
    got = orthogonalize(m).double().reshape(-1, *shape[-2:])
    for i, one in enumerate(m.reshape(-1, *shape[-2:])):
        ref, off = reference(one, 5, USUAL)
        assert float((got[i] - ref).norm()) <= off + 2.0 ** -24 * float(ref.norm()), (i, float((got[i] - ref).norm()), off)
        # elements are about wide^-1/2: one of a tile that was left out or written twice would be off by as much
        assert float((got[i] - ref).abs().max()) <= 0.05 * max(shape[-2:]) ** -0.5
