"""A residual block over node, point or token features, on the dense operators: x + W2 act(W1 norm(x) + b1) + b2, for training, and with its weights and
the features it multiplies them with in 8 bits for inference."""
from __future__ import annotations

import torch
from torch import nn

from ..operators.linear import linear_act, linear_q8
from ..operators.norm import quantize_rows, rms_norm, rms_norm_q8


class ResidualBlock(nn.Module):
    """x [..., dim] -> x + W2 act(W1 norm(x) + b1) + b2: a norm and two products, each of which reads and writes the features once.  forward takes a second
    array `residual`, whose sum with x the block then starts from (the addition is the norm's)."""

    def __init__(self, dim, hidden=None, activation="gelu", eps=1e-6, dtype=None, device=None):
        super().__init__()
        hidden = 4 * dim if hidden is None else hidden
        kw = dict(dtype=dtype, device=device)
        self.dim, self.hidden, self.activation, self.eps = dim, hidden, activation, eps
        self.norm = nn.Parameter(torch.ones(dim, **kw))
        self.w1, self.b1 = nn.Parameter(torch.empty(hidden, dim, **kw)), nn.Parameter(torch.zeros(hidden, **kw))
        self.w2, self.b2 = nn.Parameter(torch.empty(dim, hidden, **kw)), nn.Parameter(torch.zeros(dim, **kw))
        for w in (self.w1, self.w2):
            nn.init.xavier_normal_(w)

    def matrices(self):
        """The weights that an orthogonalised update (train/muon.py) is for."""
        return [self.w1, self.w2]

    def forward(self, x, residual=None):
        if residual is None:
            y, h = rms_norm(x, self.norm, eps=self.eps), x
        else:
            y, h = rms_norm(x, self.norm, residual=residual, eps=self.eps)
        u = linear_act(y, self.w1, self.b1, activation=self.activation)
        return linear_act(u, self.w2, self.b2, residual=h)

    def quantized(self, dtype=torch.int8):
        """The block for inference: weights in 8 bits, laid out once."""
        return QuantizedResidualBlock(self, dtype)


class QuantizedResidualBlock(nn.Module):
    """A ResidualBlock whose two products take operands in 8 bits (torch.int8 or torch.float8_e4m3fn) with a scale a row.  The features between blocks, the
    bias and what is added are in the type of the features, and follow the module's conversions to another."""

    def __init__(self, block, dtype=torch.int8):
        super().__init__()
        self.activation, self.eps, self.eight = block.activation, block.eps, dtype
        for name in ("norm", "b1", "b2"):
            self.register_buffer(name, getattr(block, name).detach().clone())
        for name in ("w1", "w2"):
            q, scale = quantize_rows(getattr(block, name).detach(), dtype)
            self.register_buffer(name, q)
            self.register_buffer(name + "_scale", scale)

    def _apply(self, fn, recurse=True):
        # .half(), .to(dtype): the norm's weights and the bias follow the features, what is laid out in 8 bits and its scales stay as they are
        laid_out = {name: getattr(self, name) for name in ("w1", "w1_scale", "w2", "w2_scale")}
        super()._apply(fn, recurse)
        for name, t in laid_out.items():
            if getattr(self, name).dtype is not t.dtype:
                setattr(self, name, t.to(getattr(self, name).device))
        return self

    @torch.no_grad()
    def forward(self, x, residual=None):
        if residual is None:
            (q, scale), h = rms_norm_q8(x, self.norm, eps=self.eps, dtype=self.eight), x
        else:
            q, scale, h = rms_norm_q8(x, self.norm, residual=residual, eps=self.eps, dtype=self.eight)
        u = linear_q8(q, scale, self.w1, self.w1_scale, self.b1, activation=self.activation, dtype=x.dtype)
        q, scale = quantize_rows(u, self.eight)
        return linear_q8(q, scale, self.w2, self.w2_scale, self.b2, residual=h, dtype=x.dtype)
