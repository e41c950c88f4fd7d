"""Linear maps with bias, activation and residual in the product's epilogue, and the same over operands in 8 bits: csrc/fgnn_linear.hip."""
from __future__ import annotations

import torch

from .._lib import FgnnError, dense

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3, "leaky_relu": 4}


def _activation(who, activation):
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise FgnnError("%s: activation %r; %s are supported" % (who, activation, ", ".join(str(a) for a in ACTIVATIONS)))
    return act


def linear_act(x, weight, bias=None, residual=None, activation=None, negative_slope=0.2):
    """act(x weight^T + bias) + residual for x [..., k], weight [n, k]: one pass over the result.  activation: None, "relu", "gelu" (by the error
    function), "silu" or "leaky_relu" (with negative_slope).  fp32, bf16 or fp16, the same for x, weight and residual under autocast too (bias of that type or fp32),
    sums in 32 bits; fp32 products are formed from parts of 8 significant bits, to fp32's accuracy for operands from 2^-110 on.
    Gradients of x, weight, bias and residual; those of second order are not recorded, and calls are refused in forward mode and by jit.trace, make_fx and export.
    The backward pass reads the activation's argument as rounded to the rows' type (where that is 0, relu's slope is 0) and rounds the argument's gradient to it before
    the two products; the bias gradient is summed before that.  For 16-bit rows gradients are off by about 1.4 roundings of the exact result."""
    return dense().linear_act(x, weight, bias, residual, _activation("linear_act", activation), negative_slope)


def linear_q8(q, scale, weight_q, weight_scale, bias=None, residual=None, activation=None, negative_slope=0.2, dtype=torch.bfloat16):
    """act((q * scale) (weight_q * weight_scale)^T + bias) + residual in `dtype`, for q [..., k] and weight_q [n, k] both int8 or both float8_e4m3fn, with fp32
    scales a row (as rms_norm_q8 and quantize_rows give them).  bias: of dtype or fp32; residual: of dtype.  For inference: no gradient."""
    return dense().linear_q8(q, scale, weight_q, weight_scale, bias, residual, _activation("linear_q8", activation), negative_slope, dtype)
