"""The dense operators at the ends of their ranges: long rows and row strides, small and large values, sums of integers, what they refuse."""
import pytest
import torch

from ae_mlsys_gnn_amd import _lib
from ae_mlsys_gnn_amd.operators import linear_act

from .test_linear_gpu import allowance, within

F32, BF16, F16, I8, E4M3 = range(5)


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
