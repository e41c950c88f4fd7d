"""Rows of a table by tokens, scaled, and the table's gradient by sorted tokens: csrc/fgnn_embedding.hip."""
from __future__ import annotations

from .._lib import dense


def embedding(tokens, weight, scale=1.0, padding=None):
    """scale * weight[tokens] for tokens of any shape (int32 or int64) and weight [vocabulary, channels] in fp32, bf16 or fp16.  A token outside [0, vocabulary) reads
    nothing: its row is NaN, and it gives no gradient.  The gradient of weight is dense, summed in 32 bits in the tokens' order; the row of the token
    `padding` gets none.  Gradients of second order are not recorded, and calls are refused in forward mode and by jit.trace, make_fx and export."""
    return dense().embedding(tokens, weight, scale, padding)
