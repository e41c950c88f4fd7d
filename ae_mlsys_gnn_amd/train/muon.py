"""Momentum with orthogonalised updates (Muon) for weight matrices, on the Newton-Schulz operator."""
from __future__ import annotations

import torch

from .._lib import FgnnError
from ..operators.newton_schulz import COEFFICIENTS, orthogonalize


class Muon(torch.optim.Optimizer):
    """For matrices [rows, columns]: b <- momentum b + g, then w <- (1 - lr weight_decay) w - lr max(1, rows / columns)^0.5 O, where O is g + momentum b (b without
    `nesterov`) orthogonalised.  Matrices of the same shape and type go through the same launches.  Vectors and scalars belong to another optimizer."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=coefficients))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise FgnnError("Muon: a parameter of shape %s is no matrix" % (tuple(p.shape),))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is not None:
                    alike.setdefault((tuple(p.shape), p.dtype, p.device), []).append(p)
            for (shape, _, _), ps in alike.items():
                grads = [p.grad for p in ps]
                for p in ps:
                    if "momentum" not in self.state[p]:
                        self.state[p]["momentum"] = torch.zeros_like(p)
                kept = [self.state[p]["momentum"] for p in ps]
                torch._foreach_mul_(kept, group["momentum"])
                torch._foreach_add_(kept, grads)
                updates = torch._foreach_add(grads, kept, alpha=group["momentum"]) if group["nesterov"] else kept
                out = orthogonalize(torch.stack(updates), steps=group["steps"], coefficients=group["coefficients"])
                if group["weight_decay"]:
                    torch._foreach_mul_(ps, 1.0 - group["lr"] * group["weight_decay"])
                torch._foreach_add_(ps, list(out.unbind(0)), alpha=-group["lr"] * max(1.0, shape[0] / shape[1]) ** 0.5)
        return loss
