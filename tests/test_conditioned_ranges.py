"""The conditioned blocks' operators where sizes, values and calls are out of the ordinary."""
import pytest
import torch

from . import test_group_norm_gpu as norm


@pytest.mark.gpu
@pytest.mark.parametrize("channels,dtype", [(261121, torch.float32), (262146, torch.float32), (522241, torch.bfloat16), (522247, torch.float16)])
@pytest.mark.parametrize("points", [1, 2])
def test_rows_whose_last_part_is_less_than_a_vector(channels, dtype, points):
    """Rows that workgroups share, with one to seven channels left for the last of them."""
    x, w, b, gy = norm.inputs((2, points, channels), channels, dtype, points)
    norm.check(x, 1, w, b, gy, "silu")
