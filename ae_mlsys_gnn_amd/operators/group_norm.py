"""Group norm with an activation over channels-last features: csrc/fgnn_groupnorm.hip."""
from __future__ import annotations

from .._lib import dense
from .linear import _activation


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, negative_slope=0.2):
    """act((x - mean) (var + eps)^-1/2 weight + bias) for x [samples, ..., channels], mean and (biased) variance over all points and the channels of a group of one
    sample.  weight, bias [channels] of the features' type or fp32 (None: ones, zeros); activation as of linear_act.  fp32, bf16 or fp16, with sums in 32 bits
    and more.  Points may be strided; channels that are not contiguous are copied.  Gradients of x, weight and bias, in one order of summation; those of second order
    are not recorded, and calls are refused in forward mode and by jit.trace, make_fx and export."""
    return dense().group_norm(x, groups, weight, bias, eps, _activation("group_norm", activation), negative_slope)
