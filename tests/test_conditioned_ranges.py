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
