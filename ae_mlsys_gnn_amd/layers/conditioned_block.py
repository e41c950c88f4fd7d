"""A block that brings the states of an encoder into the features of points, nodes or tokens, and the states of tokens: group norm, products, attention and embedding
of the operators package."""
from __future__ import annotations

import torch
from torch import nn

from .._lib import FgnnError
from ..operators.attention import cross_attention
from ..operators.embedding import embedding
from ..operators.group_norm import group_norm
from ..operators.linear import linear_act


class TokenStates(nn.Module):
    """tokens [samples, length] -> states [samples, length, dim], the rows of a table times dim^1/2; the row of `padding` is not trained."""

    def __init__(self, vocabulary, dim, padding=None, dtype=None, device=None):
        super().__init__()
        self.padding, self.scale = padding, dim ** 0.5
        self.table = nn.Parameter(torch.empty(vocabulary, dim, dtype=dtype, device=device))
        nn.init.normal_(self.table, std=dim ** -0.5)

    def forward(self, tokens):
        return embedding(tokens, self.table, scale=self.scale, padding=self.padding)


class ConditionedBlock(nn.Module):
    """x [samples, points, dim], states [samples, length, state_dim] -> x + Wo attention(Wq act(norm(x)), Wk states, Wv states) + bo, the norm over `groups` groups of
    channels of a sample.  kv_heads: heads of keys and values (None: heads).  forward takes which states are seen, as cross_attention does."""

    def __init__(self, dim, state_dim, heads, kv_heads=None, groups=32, activation="silu", eps=1e-5, dtype=None, device=None):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if dim % heads or heads % kv_heads or dim % groups:
            raise FgnnError("ConditionedBlock: %d features in %d heads over %d of keys, %d groups" % (dim, heads, kv_heads, groups))
        kw = dict(dtype=dtype, device=device)
        self.heads, self.kv_heads, self.width, self.groups, self.activation, self.eps = heads, kv_heads, dim // heads, groups, activation, eps
        self.norm, self.norm_bias = nn.Parameter(torch.ones(dim, **kw)), nn.Parameter(torch.zeros(dim, **kw))
        self.wq, self.wkv, self.wo = (nn.Parameter(torch.empty(s, **kw)) for s in ((dim, dim), (2 * kv_heads * self.width, state_dim), (dim, dim)))
        self.bo = nn.Parameter(torch.zeros(dim, **kw))
        for w in self.matrices():
            nn.init.xavier_normal_(w)

    def matrices(self):
        """The weights that an orthogonalised update (train/muon.py) is for."""
        return [self.wq, self.wkv, self.wo]

    def forward(self, x, states, lengths=None, mask=None):
        y = group_norm(x, self.groups, self.norm, self.norm_bias, eps=self.eps, activation=self.activation)
        q = linear_act(y, self.wq).unflatten(-1, (self.heads, self.width))
        kv = linear_act(states, self.wkv).unflatten(-1, (2, self.kv_heads, self.width))
        a = cross_attention(q, kv[:, :, 0], kv[:, :, 1], lengths=lengths, mask=mask)
        return linear_act(a.flatten(2), self.wo, self.bo, residual=x)
