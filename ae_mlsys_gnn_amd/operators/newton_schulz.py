"""Orthogonalised updates of weight matrices by Newton-Schulz products: csrc/fgnn_orth.hip."""
from __future__ import annotations

from .._lib import FgnnError, dense

# published with the Muon optimizer (K. Jordan and others, "Muon: an optimizer for hidden layers in neural networks", 2024)
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The singular values of g [..., m, n] (fp32, bf16 or fp16) moved towards one, its singular vectors kept: X = g / (|g| + eps), then `steps` times
    X <- a X + b (X X^T) X + c (X X^T)^2 X.  coefficients: (a, b, c), or one such triple for every step.  All matrices of a batch go through the same
    launches.  X and the matrices formed of it are kept to 22 significant bits, sums to 32, also for fp32; a step multiplies what small singular values
    are off by, by a.  No gradient."""
    steps = int(steps)
    try:
        flat = [float(v) for c in (coefficients if hasattr(coefficients[0], "__len__") else [coefficients] * steps) for v in c]
    except (TypeError, IndexError, ValueError):
        flat = []
    if steps < 1 or len(flat) != 3 * steps:
        raise FgnnError("orthogonalize: %d steps with coefficients %r" % (steps, coefficients))
    return dense().orthogonalize(g, flat, eps)
