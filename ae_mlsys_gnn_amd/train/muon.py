"""Momentum with orthogonalised updates (Muon) for weight matrices, on the Newton-Schulz operator."""
from __future__ import annotations

import torch

from .._lib import FgnnError
from ..operators.newton_schulz import COEFFICIENTS, orthogonalize


class Muon(torch.optim.Optimizer):
    """For matrices [rows, columns]: b <- momentum b + g, then w <- (1 - lr weight_decay) w - lr max(1, rows / columns)^0.5 O, where O is g + momentum b (b without
    `nesterov`) orthogonalised.  Matrices of the same shape and type go through the same launches.  Vectors and scalars belong to another optimizer.
    States are 32 bits.  bf16 and fp16 matrices have 32-bit weights among them, of which the parameter is the rounded form: updates and decay below its own step add
    up there.  A parameter that something else has changed is taken as it is, element by element."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=COEFFICIENTS):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=coefficients))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2:
                del self.param_groups[-1]
                raise FgnnError("Muon: a parameter of shape %s is no matrix" % (tuple(p.shape),))
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                del self.param_groups[-1]
                raise FgnnError("Muon: a parameter of %s; fp32, bf16 and fp16 are supported" % p.dtype)

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # torch has cast the states to the parameters' types
        names = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(names, (p for group in self.param_groups for p in group["params"])):
            saved = state_dict["state"].get(i, {})
            for name in saved.keys() & {"momentum", "weights"}:
                self.state[p][name] = saved[name].detach().to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    alike.setdefault((tuple(p.shape), p.dtype, p.device), []).append(p)
            for (shape, dtype, _), ps in alike.items():
                grads = [p.grad.float() for p in ps]
                for p in ps:
                    state = self.state[p]
                    if "momentum" not in state:
                        state["momentum"] = torch.zeros_like(p, dtype=torch.float32)
                    if dtype is not torch.float32 and "weights" not in state:
                        state["weights"] = p.detach().float()
                kept = [self.state[p]["momentum"] for p in ps]
                torch._foreach_mul_(kept, group["momentum"])
                torch._foreach_add_(kept, grads)
                updates = torch._foreach_add(grads, kept, alpha=group["momentum"]) if group["nesterov"] else kept
                out = orthogonalize(torch.stack(updates), steps=group["steps"], coefficients=group["coefficients"])
                ws = ps if dtype is torch.float32 else [self.state[p]["weights"] for p in ps]
                if ws is not ps:
                    for w, p in zip(ws, ps):
                        w.copy_(torch.where(w.to(dtype) == p, w, p.float()))
                if group["weight_decay"]:
                    torch._foreach_mul_(ws, 1.0 - group["lr"] * group["weight_decay"])
                torch._foreach_add_(ws, list(out.unbind(0)), alpha=-group["lr"] * max(1.0, shape[0] / shape[1]) ** 0.5)
                if ws is not ps:
                    for w, p in zip(ws, ps):
                        p.copy_(w)
        return loss
