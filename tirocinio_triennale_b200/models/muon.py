"""Muon: momentum updates of weight matrices, made nearly orthogonal before they are applied.

    opt = muon_with_adamw(model, lr=0.02, adam_lr=3e-4)

A matrix's update is its momentum after five Newton-Schulz steps (``ops.orthogonalize``), so that all directions of the
update count alike.  Matrices of one shape go through the steps together.  Embeddings, norms and biases have no use for
that and are left to AdamW.
"""
from __future__ import annotations

import torch

from .. import ops


class Muon(torch.optim.Optimizer):
    """``m = momentum m + g``, ``u = g + momentum m`` (or ``m`` without ``nesterov``), and then
    ``p = p (1 - lr weight_decay) - lr sqrt(max(1, height / width)) orthogonalize(u)``.

    Parameters: matrices on a CUDA device.  The momentum has the gradient's type, as in torch's own optimisers: float32 for float32 weights, which the
    trainer's are."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5):
        if not lr >= 0 or not 0 <= momentum < 1 or not weight_decay >= 0:
            raise ValueError("Muon: lr and weight_decay are not negative, momentum is from 0 to below 1")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError("Muon: every parameter is a matrix, got shape %s" % (tuple(p.shape),))

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
                    alike.setdefault((p.shape, p.grad.dtype, p.device), []).append(p)
            for (shape, _, _), params in alike.items():
                grads = [p.grad for p in params]
                for p in params:
                    if "momentum" not in self.state[p]:
                        self.state[p]["momentum"] = torch.zeros_like(p.grad)
                moments = [self.state[p]["momentum"] for p in params]
                torch._foreach_mul_(moments, group["momentum"])
                torch._foreach_add_(moments, grads)
                updates = torch._foreach_add(grads, moments, alpha=group["momentum"]) if group["nesterov"] else moments
                turned = ops.orthogonalize(torch.stack(updates), steps=group["steps"])
                if group["weight_decay"]:
                    torch._foreach_mul_(params, 1 - group["lr"] * group["weight_decay"])
                scale = group["lr"] * max(1.0, shape[0] / shape[1]) ** 0.5
                torch._foreach_add_(params, list(turned.to(params[0].dtype).unbind(0)), alpha=-scale)
        return loss


class Optimizers:
    """Several optimisers that step together.  A learning-rate scheduler takes one of ``optimizers``."""

    def __init__(self, *optimizers):
        self.optimizers = optimizers

    def zero_grad(self, set_to_none: bool = True):
        for o in self.optimizers:
            o.zero_grad(set_to_none=set_to_none)

    def step(self):
        for o in self.optimizers:
            o.step()

    def state_dict(self):
        return [o.state_dict() for o in self.optimizers]

    def load_state_dict(self, states):
        if len(states) != len(self.optimizers):
            raise ValueError("a state of %d optimisers for %d" % (len(states), len(self.optimizers)))
        for o, s in zip(self.optimizers, states):
            o.load_state_dict(s)


def muon_with_adamw(model: torch.nn.Module, lr: float = 0.02, adam_lr: float = 3e-4, momentum: float = 0.95, weight_decay: float = 0.0) -> Optimizers:
    """Muon for the matrices of ``model``'s linear layers, AdamW for everything else; one of them alone where the other has nothing."""
    matrices = {id(m.weight) for m in model.modules() if isinstance(m, torch.nn.Linear)}
    embedded = {id(m.weight) for m in model.modules() if isinstance(m, torch.nn.Embedding)}  # also where they are the output's
    matrices -= embedded
    params = list(model.parameters())
    turned, others = [p for p in params if id(p) in matrices], [p for p in params if id(p) not in matrices]
    optimizers = []
    if turned:
        optimizers.append(Muon(turned, lr=lr, momentum=momentum, weight_decay=weight_decay))
    if others:
        optimizers.append(torch.optim.AdamW(others, lr=adam_lr, weight_decay=weight_decay, fused=all(p.is_cuda for p in params)))
    return Optimizers(*optimizers)
