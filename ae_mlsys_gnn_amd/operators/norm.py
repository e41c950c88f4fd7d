"""Root-mean-square norm of rows with the residual's addition, as values or in 8 bits with a scale a row: csrc/fgnn_norm.hip."""
from __future__ import annotations

import torch

from .._lib import dense


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """y = h (mean(h^2) + eps)^-1/2 weight over the last dimension of h = x + residual: y, or (y, h) with a residual.  fp32, bf16 or fp16 rows of up to
    64 KB; weight [features] of their type or fp32 (None: ones).  Statistics are 32 bits.  Gradients of x, weight and residual; those of second order are not
    recorded, and calls are refused in forward mode and by jit.trace, make_fx and export.  y is the norm of the sum before it is rounded to h, the backward pass reads
    h: for 16-bit rows with a residual the weight's gradient is off by about 1.4 roundings of the exact result."""
    return dense().rms_norm(x, weight, residual, eps)


def rms_norm_q8(x, weight=None, residual=None, eps=1e-6, dtype=torch.int8):
    """The norm's output in 8 bits: (q, scale), or (q, scale, h) with a residual, with y = q * scale[..., None].  scale is fp32, one a row: its
    largest magnitude over 127 (int8) or 448 (float8_e4m3fn); a row with an infinity or a NaN gets the scale NaN.  For inference: no gradient."""
    return dense().rms_norm_q8(x, weight, residual, eps, dtype)


def quantize_rows(x, dtype=torch.int8):
    """Rows as they are in 8 bits: (q, scale) as of rms_norm_q8.  The weights of linear_q8 are laid out by it once."""
    return dense().quantize_rows(x, dtype)
