"""Residual blocks, their 8-bit form, the optimizer of orthogonalised updates, and the GAT driver that runs them together."""
import copy

import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.layers import ResidualBlock
from ae_mlsys_gnn_amd.train.muon import Muon

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def composed(block, x, residual=None):
    """The block in float64, from torch's operations."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in block.named_parameters()}
    h = x if residual is None else x + residual
    y = h * (h.square().mean(-1, keepdim=True) + block.eps).rsqrt() * p["norm"]
    u = torch.nn.functional.gelu(y @ p["w1"].t() + p["b1"])
    return h + u @ p["w2"].t() + p["b2"], p


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("rows,dim,hidden", [(1, 64, None), (300, 100, 41), (1000, 256, 512)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_block_and_gradients(dtype, rows, dim, hidden, with_residual):
    torch.manual_seed(rows + dim)
    block = ResidualBlock(dim, hidden).to("cuda", dtype)
    with torch.no_grad():
        for p in (block.norm, block.b1, block.b2):
            p.add_(0.2 * torch.randn_like(p))
    x, r, gy = (torch.randn(rows, dim).to(dtype) for _ in range(3))
    xl, rl = x.cuda().requires_grad_(True), r.cuda().requires_grad_(True) if with_residual else None
    out = block(xl, rl)
    out.backward(gy.cuda())
    xd, rd = x.double().requires_grad_(True), r.double().requires_grad_(True) if with_residual else None
    ref, p = composed(block, xd, rd)
    ref.backward(gy.double())

    # every value on the way is rounded to the type a handful of times (h, y, z, u; and their gradients): norm-wise 12 unit roundoffs, each at most
    # the type's; sums in 32 bits are below that for the 16-bit types and 2^-20 for fp32
    bar = max(12 * UNIT[dtype], 2.0 ** -20)
    named = dict(block.named_parameters())
    pairs = [("out", out, ref), ("x", xl.grad, xd.grad)] + [(k, named[k].grad, p[k].grad) for k in p]
    if with_residual:
        pairs.append(("residual", rl.grad, rd.grad))
    for what, got, want in pairs:
        got, want = got.detach().double().cpu(), want.detach()
        assert float((got - want).norm()) <= bar * float(want.norm()) + 1e-12, what


@pytest.mark.gpu
@pytest.mark.parametrize("eight,bar", [(torch.int8, 0.02), (torch.float8_e4m3fn, 0.08)])
@pytest.mark.parametrize("rows", [1, 17, 500])
def test_eight_bit_block(eight, bar, rows):
    # the branch's two products carry operands off by up to half a step: int8 1 / 254 of a row's maximum (about four times its mean), e4m3 2^-4 of each value
    torch.manual_seed(rows)
    block = ResidualBlock(256, 384).cuda()
    x, r = torch.randn(rows, 256).cuda(), torch.randn(rows, 256).cuda()
    served = block.quantized(eight)
    with torch.no_grad():
        for args, h in (((x,), x), ((x, r), x + r)):
            branch = block(*args) - h
            got = served(*args) - h
            assert float((got - branch).norm()) <= bar * float(branch.norm())
    assert not served(x).requires_grad and served.state_dict()["w1"].dtype is eight


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_against_float64(nesterov):
    torch.manual_seed(0)
    shapes = [(40, 64), (64, 40), (40, 64), (100, 7)]
    ws = [torch.nn.Parameter(torch.randn(s).cuda()) for s in shapes]
    ref = [w.detach().double().cpu() for w in ws]
    buf = [torch.zeros_like(w) for w in ref]
    opt = Muon(ws, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.01)
    a, b, c = 3.4445, -4.7750, 2.0315
    for step in range(3):
        for i, w in enumerate(ws):
            g = torch.randn(shapes[i])
            w.grad = g.cuda()
            buf[i] = 0.9 * buf[i] + g.double()
            u = g.double() + 0.9 * buf[i] if nesterov else buf[i]
            u = u / (u.norm() + 1e-7)
            for _ in range(5):
                gram = u @ u.t()
                u = a * u + (b * gram + c * gram @ gram) @ u
            ref[i] = ref[i] * (1 - 0.1 * 0.01) - 0.1 * max(1.0, shapes[i][0] / shapes[i][1]) ** 0.5 * u
        opt.step()
    for w, r in zip(ws, ref):
        # an update is exact to about 1e-3 in norm at the worst (22 bits times what five steps make of them), here far below
        assert float((w.detach().double().cpu() - r).norm()) <= 1e-4 * float(r.norm())
    frozen = copy.deepcopy([w.detach() for w in ws])
    opt.zero_grad()
    opt.step()
    assert all(torch.equal(w, f) for w, f in zip(ws, frozen))


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [[], ["--hip-graph"]])
def test_gat_driver_with_blocks(tmp_path, extra):
    from ae_mlsys_gnn_amd.train import train_gatconv
    common = ["--dataset", "cora", "--num-hidden", "16", "--num-heads", "2", "--epochs", "30", "--output", str(tmp_path / "o.csv"), "--scale", "0.5"]
    plain = train_gatconv.main(common)
    assert plain["test_acc_eight_bit"] is None
    out = train_gatconv.main(common + ["--residual-blocks", "2", "--optimizer", "muon", "--eight-bit", "int8"] + extra)
    assert out["last_loss"] < out["first_loss"] and out["last_loss"] == out["last_loss"]
    assert abs(out["test_acc_eight_bit"] - out["test_acc"]) < 0.1


def test_muon_refuses_vectors():
    with pytest.raises(_lib.FgnnError, match="no matrix"):
        Muon([torch.nn.Parameter(torch.randn(5))])


@pytest.mark.gpu
def test_replayed_graphs_give_what_eager_calls_give():
    from ae_mlsys_gnn_amd.operators import linear_act, linear_q8, orthogonalize, quantize_rows, rms_norm, rms_norm_q8
    torch.manual_seed(1)
    x, r, w, wide = torch.randn(700, 128).cuda(), torch.randn(700, 128).cuda(), torch.randn(96, 128).cuda(), torch.randn(3, 300, 520).cuda()
    tall = torch.randn(40000, 64, device="cuda", dtype=torch.bfloat16)
    wt = torch.randn(48, 64, device="cuda", dtype=torch.bfloat16)
    wq, ws = quantize_rows(w)
    leaf, wleaf = tall.clone().requires_grad_(True), wt.clone().requires_grad_(True)

    def work():
        y, h = rms_norm(x, None, residual=r)
        q, s = rms_norm_q8(x)
        grads = torch.autograd.grad(linear_act(leaf, wleaf, activation="silu"), (leaf, wleaf), torch.ones(40000, 48, device="cuda", dtype=torch.bfloat16))
        return (y, h, linear_act(h, w, activation="gelu"), linear_q8(q, s, wq, ws), orthogonalize(wide), orthogonalize(w)) + grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(4):
        with torch.no_grad():
            for t in (x, r, wide, leaf, wleaf):
                t.copy_(torch.randn_like(t))
        eager = [t.clone() for t in work()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i
