"""Linear maps with bias, activation and residual in the product's epilogue, and the same over operands in 8 bits: csrc/fgnn_linear.hip."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .._lib import EIGHT_TYPES, FLOAT_TYPES, FgnnError, check, device_guard, lib, ptr, require_cuda, rows_of, stream_ptr, workspace

ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "silu": 3, "leaky_relu": 4}


def _activation(who, activation):
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise FgnnError("%s: activation %r; %s are supported" % (who, activation, ", ".join(str(a) for a in ACTIVATIONS)))
    return act


def _epilogue(who, shape, n, dtype, device, bias, residual):
    """Checked (bias, its type, residual as rows, its row stride) beside an output [..., n] of dtype."""
    kind = FLOAT_TYPES[dtype]
    if bias is not None:
        if bias.shape != (n,) or bias.dtype not in (dtype, torch.float32) or bias.device != device:
            raise FgnnError("%s: bias %s of %s for %d columns of %s" % (who, tuple(bias.shape), bias.dtype, n, dtype))
        bias = bias.contiguous()
    ldr = 0
    if residual is not None:
        if residual.shape != shape[:-1] + (n,) or residual.dtype != dtype or residual.device != device:
            raise FgnnError("%s: residual %s of %s beside %s of %s" % (who, tuple(residual.shape), residual.dtype, tuple(shape[:-1]) + (n,), dtype))
        residual, ldr = rows_of(residual, who)
    return bias, kind if bias is None else FLOAT_TYPES[bias.dtype], residual, ldr


def _operands(x, weight):
    require_cuda(x, weight)
    kind = FLOAT_TYPES.get(x.dtype)
    if kind is None or weight.dtype != x.dtype:
        raise FgnnError("linear_act: rows of %s with weights of %s; fp32, bf16 and fp16, both the same, are supported" % (x.dtype, weight.dtype))
    if x.dim() == 0 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.device != x.device:
        raise FgnnError("linear_act: x %s with weights %s" % (tuple(x.shape), tuple(weight.shape)))
    return kind


def _forward(x, weight, bias, residual, act, slope, keep):
    """(y, z): z, the activation's argument, where `keep`."""
    kind = _operands(x, weight)
    shape, (n, k) = x.shape, weight.shape
    require_cuda(bias, residual)
    bias, btype, residual, ldr = _epilogue("linear_act", shape, n, x.dtype, x.device, bias, residual)
    x, ldx = rows_of(x, "linear_act")
    weight, ldw = rows_of(weight, "linear_act")
    rows = x.shape[0]
    y = torch.empty(shape[:-1] + (n,), dtype=x.dtype, device=x.device)
    z = torch.empty((rows, n), dtype=x.dtype, device=x.device) if keep else None
    with device_guard(x.device):
        ws, wsb = workspace(lib().fgnn_linear_workspace_bytes(rows, n, k, kind), x.device)
        check(lib().fgnn_linear(rows, n, k, kind, ptr(x), ldx, ptr(weight), ldw, ptr(bias), btype, ptr(residual), ldr, act, slope, ptr(z), ptr(y), ptr(ws), wsb,
                                stream_ptr()), "fgnn_linear")
    return y, z


class LinearActFunction(torch.autograd.Function):
    """y = act(x W^T + b) + r.  Kept for the backward pass: x, W and, with an activation, its argument in the rows' type."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, slope):
        y, z = _forward(x, weight, bias, residual, act, slope, act != 0)
        ctx.act, ctx.slope = act, slope
        ctx.btype = None if bias is None else bias.dtype
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        kind, dtype, device = FLOAT_TYPES[x.dtype], x.dtype, x.device
        shape, (n, k) = x.shape, weight.shape
        dx = dw = db = None
        x, ldx = rows_of(x, "linear_act")
        weight, ldw = rows_of(weight, "linear_act")
        rows = x.shape[0]
        dz, ldz = rows_of(gy, "linear_act")
        sloped = ctx.act and (need_x or need_w)
        with device_guard(device):
            stream = stream_ptr()
            if n and (sloped or need_b):
                g, ldg = dz, ldz
                if sloped:
                    dz, ldz = torch.empty((rows, n), dtype=dtype, device=device), n
                if need_b:
                    db = torch.empty(n, dtype=ctx.btype, device=device)
                ws, wsb = workspace(lib().fgnn_linear_slope_workspace_bytes(rows, n, kind) if need_b else 0, device)
                check(lib().fgnn_linear_slope(rows, n, kind, ptr(g), ldg, ptr(z), ctx.act, ctx.slope, ptr(dz) if sloped else None, ptr(db),
                                              FLOAT_TYPES[ctx.btype] if need_b else kind, ptr(ws), wsb, stream), "fgnn_linear_slope")
            if need_x or need_w:
                ws, wsb = workspace(lib().fgnn_linear_backward_workspace_bytes(rows, n, k, kind), device)
            if need_x:
                dx = torch.empty(shape, dtype=dtype, device=device)
                check(lib().fgnn_linear_dx(rows, n, k, kind, ptr(dz), ldz, ptr(weight), ldw, ptr(dx), ptr(ws), wsb, stream), "fgnn_linear_dx")
            if need_w:
                dw = torch.empty((n, k), dtype=dtype, device=device)
                check(lib().fgnn_linear_dw(rows, n, k, kind, ptr(dz), ldz, ptr(x), ldx, ptr(dw), ptr(ws), wsb, stream), "fgnn_linear_dw")
        if need_b and db is None:
            db = torch.empty(0, dtype=ctx.btype, device=device)
        return dx, dw, db, gy if need_r else None, None, None


def linear_act(x, weight, bias=None, residual=None, activation=None, negative_slope=0.2):
    """act(x weight^T + bias) + residual for x [..., k], weight [n, k]: one pass over the result.  activation: None, "relu", "gelu" (by the error
    function), "silu" or "leaky_relu" (with negative_slope).  fp32, bf16 or fp16 (bias of that type or fp32), sums in 32 bits; fp32 products are formed from
    parts of 8 significant bits to fp32's accuracy.  Gradients of x, weight, bias and residual; those of second order are not recorded."""
    act = _activation("linear_act", activation)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return LinearActFunction.apply(x, weight, bias, residual, act, float(negative_slope))
    return _forward(x, weight, bias, residual, act, float(negative_slope), False)[0]


def linear_q8(q, scale, weight_q, weight_scale, bias=None, residual=None, activation=None, negative_slope=0.2, dtype=torch.bfloat16):
    """act((q * scale) (weight_q * weight_scale)^T + bias) + residual in `dtype`, for q [..., k] and weight_q [n, k] both int8 or both float8_e4m3fn, with fp32
    scales a row (as rms_norm_q8 and quantize_rows give them).  bias: of dtype or fp32; residual: of dtype.  For inference: no gradient."""
    act = _activation("linear_q8", activation)
    require_cuda(q, scale, weight_q, weight_scale, bias, residual)
    eight = EIGHT_TYPES.get(q.dtype)
    if eight is None or weight_q.dtype != q.dtype or dtype not in FLOAT_TYPES:
        raise FgnnError("linear_q8: %s with weights of %s to %s; int8 or float8_e4m3fn, both the same, to fp32, bf16 or fp16 are supported" % (
            q.dtype, weight_q.dtype, dtype))
    if q.dim() == 0 or weight_q.dim() != 2 or weight_q.shape[1] != q.shape[-1] or scale.shape != q.shape[:-1] or weight_scale.shape != weight_q.shape[:1]:
        raise FgnnError("linear_q8: q %s, scale %s, weights %s, their scale %s" % (tuple(q.shape), tuple(scale.shape), tuple(weight_q.shape), tuple(weight_scale.shape)))
    if not (scale.dtype is weight_scale.dtype is torch.float32) or not q.device == scale.device == weight_q.device == weight_scale.device:
        raise FgnnError("linear_q8: scales are fp32 on the operands' device")
    shape, (n, k), kind = q.shape, weight_q.shape, FLOAT_TYPES[dtype]
    bias, btype, residual, ldr = _epilogue("linear_q8", shape, n, dtype, q.device, bias, residual)
    q, ldq = rows_of(q, "linear_q8")
    weight_q, ldw = rows_of(weight_q, "linear_q8")
    scale, weight_scale = scale.contiguous(), weight_scale.contiguous()
    rows = q.shape[0]
    y = torch.empty(shape[:-1] + (n,), dtype=dtype, device=q.device)
    with device_guard(q.device):
        ws, wsb = workspace(lib().fgnn_linear_workspace_bytes(rows, n, k, eight), q.device)
        check(lib().fgnn_linear_q8(rows, n, k, eight, kind, ptr(q), ldq, ptr(scale), ptr(weight_q), ldw, ptr(weight_scale), ptr(bias), btype, ptr(residual), ldr,
                                   act, float(negative_slope), ptr(y), ptr(ws), wsb, stream_ptr()), "fgnn_linear_q8")
    return y
