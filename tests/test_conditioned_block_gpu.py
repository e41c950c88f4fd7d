"""Blocks that bring an encoder's states into features, the states of tokens, and the point-cloud driver that runs them together."""
import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.layers import ConditionedBlock, ResidualBlock, TokenStates

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def composed(block, states, x, tokens, mask, fixed=False):
    """Both modules in float64, from torch's operations.  fixed: the softmax's sums are taken as constants, so that the gradient of a score is P dP alone."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in list(block.named_parameters()) + list(states.named_parameters())}
    b, n, dim = x.shape
    h, hk, d = block.heads, block.kv_heads, block.width
    y = torch.nn.functional.silu(torch.nn.functional.group_norm(x.transpose(1, 2), block.groups, p["norm"], p["norm_bias"], block.eps)).transpose(1, 2)
    e = p["table"][tokens] * states.scale
    q = (y @ p["wq"].t()).view(b, n, h, d).transpose(1, 2)
    kv = (e @ p["wkv"].t()).view(b, -1, 2, hk, d)
    k, v = (kv[:, :, i].transpose(1, 2).repeat_interleave(h // hk, 1) for i in range(2))
    s = (q @ k.transpose(2, 3) / d ** 0.5).masked_fill(~mask.view(b, 1, 1, -1), -torch.inf)
    w = torch.softmax(s, -1).nan_to_num(0.0)
    if fixed:
        w = w.detach() * torch.exp(s - s.detach()).nan_to_num(0.0)
    a = w @ v
    return x + a.transpose(1, 2).reshape(b, n, dim) @ p["wo"].t() + p["bo"], p


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(UNIT))
@pytest.mark.parametrize("batch,points,dim,heads,kv_heads,length", [(2, 100, 64, 4, 2, 17), (1, 1, 96, 3, 3, 1), (3, 257, 128, 2, 1, 70)])
def test_block_and_gradients(dtype, batch, points, dim, heads, kv_heads, length):
    torch.manual_seed(points + dim)
    block = ConditionedBlock(dim, 40, heads, kv_heads, groups=8).to("cuda", dtype)
    states = TokenStates(50, 40, padding=0).to("cuda", dtype)
    with torch.no_grad():
        for p in (block.norm, block.norm_bias, block.bo):
            p.add_(0.2 * torch.randn_like(p))
    x, gy = torch.randn(batch, points, dim).to(dtype), torch.randn(batch, points, dim).to(dtype)
    tokens, mask = torch.randint(1, 50, (batch, length)), torch.rand(batch, length) < 0.7
    mask[:, 0] = True
    tokens[~mask] = 0
    if batch > 2:
        mask[2] = False                     # a sample without states keeps its features, but for the bias
    xl = x.cuda().requires_grad_(True)
    out = block(xl, states(tokens.cuda()), mask=mask.cuda())
    out.backward(gy.cuda())
    xd = x.double().requires_grad_(True)
    ref, p = composed(block, states, xd, tokens, mask)
    ref.backward(gy.double())
    # A score's gradient P dP - P delta is the difference of two terms that are each off by their own roundings, and cancel where a sample sees one state (P = 1, delta = dP: the
    # exact gradient is 0). All else is linear in it: a gradient is off by its roundings times the size of the first term's share plus that of the second's, which
    # is the first's less the gradient.
    xf = x.double().requires_grad_(True)
    first, pf = composed(block, states, xf, tokens, mask, fixed=True)
    first.backward(gy.double())
    # about a dozen roundings to the type lie one behind the other (norm, q, states, k and v, weights, attention, and their gradients): norm-wise 24 unit
    # roundoffs, each at most the type's; for fp32 sums in 32 bits, 2^-18
    bar = max(24 * UNIT[dtype], 2.0 ** -18)
    named = dict(list(block.named_parameters()) + list(states.named_parameters()))
    for what, got, want, one in [("out", out, ref, first), ("x", xl.grad, xd.grad, xf.grad)] + [(k, named[k].grad, p[k].grad, pf[k].grad) for k in p]:
        got, want, one = got.detach().double().cpu(), want.detach(), one.detach()
        if what == "table":                 # (the padding's row has no gradient)
            got, want, one = got[1:], want[1:], one[1:]
        assert float((got - want).norm()) <= bar * float(torch.maximum(want.norm(), one.norm() + (one - want).norm())) + 1e-9, what
    assert (named["table"].grad[0] == 0).all()


@pytest.mark.gpu
def test_a_run_of_blocks_by_lengths_and_single_points():
    torch.manual_seed(0)
    block, states, res = ConditionedBlock(128, 64, 4, 2).cuda(), TokenStates(30, 64).cuda(), ResidualBlock(128).cuda()
    tokens, lengths = torch.randint(0, 30, (4, 25)).cuda(), torch.tensor([25, 1, 0, 13]).cuda()
    x = torch.randn(4, 60, 128).cuda()
    e = states(tokens)
    out = res(block(x, e, lengths=lengths))
    same = res(block(x, e, mask=torch.arange(25).cuda() < lengths[:, None]))
    assert torch.equal(out, same) and torch.isfinite(out).all()
    loss = (out * torch.randn_like(out)).sum()
    grads = torch.autograd.grad(loss, list(block.parameters()) + list(states.parameters()) + list(res.parameters()))
    assert all(torch.isfinite(g).all() and (g != 0).any() for g in grads)
    with torch.no_grad():                   # one point at a time, for inference
        one = block(x[:, :1].contiguous(), e, lengths=lengths)
        assert one.shape == (4, 1, 128) and torch.allclose(one[2], x[2, :1] + block.bo)


@pytest.mark.gpu
def test_point_cloud_driver_with_norm_and_voxels(tmp_path):
    from ae_mlsys_gnn_amd.train import train_edgeconv
    common = ["--num-clouds", "40", "--num-points", "128", "--batch-size", "8", "--k", "8", "--num-epochs", "2", "--warmup-epochs", "1", "--iters-per-epoch", "2",
              "--output", str(tmp_path / "o.csv")]
    out = train_edgeconv.main(common + ["--norm-groups", "16", "--voxel-tokens", "32", "--heads", "4"])
    assert len(out["losses"]) == 3 and all(l == l for l in out["losses"])
    out = train_edgeconv.main(common + ["--voxel-tokens", "500"])       # more than the cloud has points
    assert all(l == l for l in out["losses"])


@pytest.mark.gpu
def test_gradients_of_the_driver_model():
    from ae_mlsys_gnn_amd.train.train_edgeconv import Model
    torch.manual_seed(0)
    model = Model(4, [64, 64], [512, 128], 5, norm_groups=32, tokens=20, grid=4).cuda()
    loss = model(torch.rand(3, 64, 3).cuda()).square().sum()
    loss.backward()
    for name, p in model.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    assert all((p.grad != 0).any() for p in [model.norm, model.norm_bias, model.states.table] + model.condition.matrices())


def test_voxel_tokens():
    from ae_mlsys_gnn_amd.train.train_edgeconv import voxel_tokens
    x = torch.rand(3, 50, 3, generator=torch.Generator().manual_seed(0)) * 4 - 1
    tokens, seen = voxel_tokens(x, 20, 4)
    assert tokens.shape == seen.shape == (3, 20) and tokens.min() >= 0 and tokens.max() < 64
    for b in range(3):
        box = (x[b] - x[b].min(0).values) / (x[b].max(0).values - x[b].min(0).values)
        cells = {int(a) * 16 + int(c) * 4 + int(d) for a, c, d in (box[:20] * 4).long().clamp(0, 3).tolist()}
        assert sorted(cells) == tokens[b][seen[b]].tolist()
    flat, _ = voxel_tokens(torch.zeros(1, 5, 3), 5, 4)
    assert (flat == 0).all()


def test_driver_refusals():
    from ae_mlsys_gnn_amd.train import train_edgeconv
    for bad in (["--norm-groups", "7"], ["--voxel-tokens", "-1"], ["--heads", "3"], ["--heads", "1"], ["--voxel-grid", "0"]):
        with pytest.raises(SystemExit):
            train_edgeconv.main(bad)
    with pytest.raises(_lib.FgnnError, match="heads"):
        ConditionedBlock(64, 8, 3)
