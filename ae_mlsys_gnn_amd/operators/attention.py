"""Attention of one set of features to the states of another, of its own length: csrc/fgnn_attention.h."""
from __future__ import annotations

from .._lib import dense


def cross_attention(q, k, v, lengths=None, mask=None, scale=None):
    """softmax(scale q k^T) v for queries q [samples, queries, heads, components] over keys and values k, v [samples, keys, kv_heads, components], where head h uses the
    keys of head h // (heads / kv_heads); components <= 256; scale None: components^-1/2.  A sample's queries see its first lengths[sample] keys (int32 or int64, cut
    to 0 .. keys; None: all), and of them those with mask[sample, key] (bool; None: all).  Queries that see no key get zeros and no gradient; what lies in keys and
    values that are not seen is never used, NaN neither, and their gradient is 0.
    fp32, bf16 or fp16, the same for q, k and v, of any strides (components that are not contiguous are copied).  Sums, softmax and results are 32 bits; of 16-bit
    types the softmax's weights and the scores' gradient are rounded to the type before they are multiplied, and a call that trains q or k keeps what the rounding of its
    results leaves, as much memory again, for their gradients.  Products of fp32 are formed from parts of 8 significant bits, as near to float64 as fp32 products are, and an
    infinity in keys or values that are seen, or in queries, gives NaN there.  Gradients of q, k and v, in one order of summation; calls that train k or v are refused for
    samples x kv_heads x ceil(keys / 128) of 2^24 and more.  Gradients of second order are not recorded, and calls are refused in forward mode and by jit.trace, make_fx and
    export."""
    return dense().cross_attention(q, k, v, lengths, mask, scale)
