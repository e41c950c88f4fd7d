"""Root-mean-square norm of rows with the residual's addition, as values or in 8 bits with a scale a row: csrc/fgnn_norm.hip."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .._lib import EIGHT_TYPES, FLOAT_TYPES, FgnnError, check, device_guard, lib, ptr, require_cuda, rows_of, stream_ptr, workspace


def _operands(who, x, weight, residual):
    """Checked operands as (x, its row stride, residual, its row stride, weight, the types' codes)."""
    require_cuda(x, weight, residual)
    kind = FLOAT_TYPES.get(x.dtype)
    if kind is None:
        raise FgnnError("%s: rows of %s; fp32, bf16 and fp16 are supported" % (who, x.dtype))
    if x.dim() == 0 or x.shape[-1] == 0:
        raise FgnnError("%s: no features in %s" % (who, tuple(x.shape)))
    wkind = kind
    if weight is not None:
        if weight.shape != x.shape[-1:] or weight.dtype not in (x.dtype, torch.float32) or weight.device != x.device:
            raise FgnnError("%s: weights %s of %s for rows %s of %s" % (who, tuple(weight.shape), weight.dtype, tuple(x.shape), x.dtype))
        weight = weight.contiguous()
        wkind = FLOAT_TYPES[weight.dtype]
    r, ldr = None, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device:
            raise FgnnError("%s: residual %s of %s beside %s of %s" % (who, tuple(residual.shape), residual.dtype, tuple(x.shape), x.dtype))
        r, ldr = rows_of(residual, who)
    x, ldx = rows_of(x, who)
    return x, ldx, r, ldr, weight, kind, wkind


def _forward(x, weight, residual, eps, want_rstd):
    shape = x.shape
    x, ldx, r, ldr, weight, kind, wkind = _operands("rms_norm", x, weight, residual)
    rows, cols = x.shape
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    h = torch.empty(shape, dtype=x.dtype, device=x.device) if r is not None else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_rstd else None
    with device_guard(x.device):
        check(lib().fgnn_rms_norm(rows, cols, kind, ptr(x), ldx, ptr(r), ldr, ptr(weight), wkind, eps, ptr(h), ptr(y), ptr(rstd), stream_ptr()), "fgnn_rms_norm")
    return y, h, rstd


class RMSNormFunction(torch.autograd.Function):
    """y (and h = x + residual).  Kept for the backward pass: h as it is handed out (x without a residual) and a scale a row; the norm itself is taken
    of the sum before it is rounded."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = _forward(x, weight, residual, eps, True)
        ctx.set_materialize_grads(False)
        ctx.with_residual = residual is not None
        ctx.save_for_backward(x if h is None else h, weight, rstd)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gh=None):
        h, weight, rstd = ctx.saved_tensors
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if gy is None and gh is None or not (need_x or need_w or need_r):
            return None, None, None, None
        shape = h.shape
        h, ldh = rows_of(h, "rms_norm")
        rows, cols = h.shape
        kind = FLOAT_TYPES[h.dtype]
        gy = None if gy is None else gy.contiguous()
        gh = None if gh is None else gh.contiguous()
        dx = torch.empty(shape, dtype=h.dtype, device=h.device) if need_x or need_r else None
        weight = None if weight is None else weight.contiguous()
        dw = torch.empty_like(weight) if need_w else None
        with device_guard(h.device):
            ws, wsb = workspace(lib().fgnn_rms_norm_backward_workspace_bytes(rows, cols, kind) if need_w else 0, h.device)
            check(lib().fgnn_rms_norm_backward(rows, cols, kind, ptr(gy), ptr(gh), ptr(h), ldh, ptr(weight), kind if weight is None else FLOAT_TYPES[weight.dtype],
                                               ptr(rstd), ptr(dx), ptr(dw), ptr(ws), wsb, stream_ptr()), "fgnn_rms_norm_backward")
        return dx if need_x else None, dw, dx if need_r else None, None


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """y = h (mean(h^2) + eps)^-1/2 weight over the last dimension of h = x + residual: y, or (y, h) with a residual.  fp32, bf16 or fp16 rows of up to
    64 KB; weight [features] of their type or fp32 (None: ones).  Statistics are 32 bits."""
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (residual is not None and residual.requires_grad)):
        return RMSNormFunction.apply(x, weight, residual, float(eps))
    y, h, _ = _forward(x, weight, residual, float(eps), False)
    return y if h is None else (y, h)


def _eight(who, dtype):
    kind = EIGHT_TYPES.get(dtype)
    if kind is None:
        raise FgnnError("%s: 8-bit output in %s; torch.int8 and torch.float8_e4m3fn are supported" % (who, dtype))
    return kind


def rms_norm_q8(x, weight=None, residual=None, eps=1e-6, dtype=torch.int8):
    """The norm's output in 8 bits: (q, scale), or (q, scale, h) with a residual, with y = q * scale[..., None].  scale is fp32, one a row: its
    largest magnitude over 127 (int8) or 448 (float8_e4m3fn); a row with an infinity or a NaN gets the scale NaN.  For inference: no gradient."""
    shape, eight = x.shape, _eight("rms_norm_q8", dtype)
    x, ldx, r, ldr, weight, kind, wkind = _operands("rms_norm_q8", x, weight, residual)
    q = torch.empty(shape, dtype=dtype, device=x.device)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    h = torch.empty(shape, dtype=x.dtype, device=x.device) if r is not None else None
    with device_guard(x.device):
        check(lib().fgnn_rms_norm_q8(x.shape[0], x.shape[1], kind, ptr(x), ldx, ptr(r), ldr, ptr(weight), wkind, float(eps), eight, ptr(h), ptr(q), ptr(scale),
                                     stream_ptr()), "fgnn_rms_norm_q8")
    return (q, scale) if h is None else (q, scale, h)


def quantize_rows(x, dtype=torch.int8):
    """Rows as they are in 8 bits: (q, scale) as of rms_norm_q8.  The weights of linear_q8 are laid out by it once."""
    shape, eight = x.shape, _eight("quantize_rows", dtype)
    x, ldx, _, _, _, kind, _ = _operands("quantize_rows", x, None, None)
    q = torch.empty(shape, dtype=dtype, device=x.device)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    with device_guard(x.device):
        check(lib().fgnn_quantize_rows(x.shape[0], x.shape[1], kind, ptr(x), ldx, eight, ptr(q), ptr(scale), stream_ptr()), "fgnn_quantize_rows")
    return q, scale
