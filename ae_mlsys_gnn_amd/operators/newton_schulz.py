"""Orthogonalised updates of weight matrices by Newton-Schulz products: csrc/fgnn_orth.hip."""
from __future__ import annotations

import ctypes

import torch

from .._lib import FLOAT_TYPES, FgnnError, check, device_guard, lib, ptr, require_cuda, stream_ptr, workspace

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The singular values of g [..., m, n] (fp32, bf16 or fp16) moved towards one, its singular vectors kept: X = g / (|g| + eps), then `steps` times
    X <- a X + b (X X^T) X + c (X X^T)^2 X.  coefficients: (a, b, c), or one such triple for every step.  All matrices of a batch go through the same
    launches.  The products carry 22 significant bits and sums 32, so the result is that of fp32.  No gradient."""
    require_cuda(g)
    kind = FLOAT_TYPES.get(g.dtype)
    if kind is None or g.dim() < 2:
        raise FgnnError("orthogonalize: matrices %s of %s; fp32, bf16 and fp16 are supported" % (tuple(g.shape), g.dtype))
    steps = int(steps)
    try:
        flat = [float(v) for c in (coefficients if hasattr(coefficients[0], "__len__") else [coefficients] * steps) for v in c]
    except (TypeError, IndexError, ValueError):
        flat = []
    if steps < 1 or len(flat) != 3 * steps:
        raise FgnnError("orthogonalize: %d steps with coefficients %r" % (steps, coefficients))
    g = g.detach().contiguous()
    m, n = g.shape[-2:]
    batch = g.shape[:-2].numel()
    out = torch.empty_like(g)
    with device_guard(g.device):
        ws, wsb = workspace(lib().fgnn_orthogonalize_workspace_bytes(batch, m, n), g.device)
        check(lib().fgnn_orthogonalize(batch, m, n, kind, ptr(g), steps, (ctypes.c_float * (3 * steps))(*flat), float(eps), ptr(out), ptr(ws), wsb, stream_ptr()),
              "fgnn_orthogonalize")
    return out
