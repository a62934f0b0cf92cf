"""AdamW whose step is one launch over all tensors of a parameter group (``ops.adamw_step``), with moments in 32 or in 8 bits.

    opt = AdamW(model.parameters(), lr=3e-4, bits=8)

Moments in 8 bits take 2.06 bytes a parameter instead of 8.
"""
from __future__ import annotations

import torch

from .. import ops
from ..ops.adamw import BLOCK


class AdamW(torch.optim.Optimizer):
    """The update of ``ops.adamw_step``.  Parameters: CUDA tensors without gaps, float32, bfloat16 or float16.

    ``bits``: 32, or 8 for moments of a byte each with a scale for every 256 of them; ``seed``: of their random rounding.
    ``capturable``: the step's number is held on the device and counted for a group as a whole, so that a captured step can be replayed; ``lr`` may
    then be a float32 CUDA tensor of one value, which can be changed between replays.  A step that is captured without it, or that comes before every parameter's state
    has begun in a step outside, raises RuntimeError."""

    def __init__(self, params, lr: float | torch.Tensor = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, bits: int = 32, seed: int = 0,
                 capturable: bool = False):
        if not isinstance(lr, torch.Tensor) and not lr >= 0 or not 0 <= betas[0] < 1 or not 0 <= betas[1] < 1 or not eps >= 0 or not weight_decay >= 0:
            raise ValueError("AdamW: lr, eps and weight_decay are not negative, betas are from 0 to below 1")
        if bits not in (8, 32):
            raise ValueError("AdamW: moments are held in 8 or in 32 bits, got %r" % (bits,))
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits, seed=seed, capturable=capturable))

    def _begin(self, p, bits):
        like = torch.uint8 if bits == 8 else torch.float32
        state = {"exp_avg": torch.zeros_like(p, dtype=like), "exp_avg_sq": torch.zeros_like(p, dtype=like)}
        if bits == 8:
            state["scales"] = torch.zeros((p.numel() + BLOCK - 1) // BLOCK, 2, device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_current_stream_capturing():
            self._check_capture()
        for number, group in enumerate(self.param_groups):
            alike = {}  # a parameter that had no gradient in some step is behind the others
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    state.update(self._begin(p, group["bits"]))
                    if not group["capturable"]:
                        state["step"] = 0
                if not group["capturable"]:
                    state["step"] += 1
                alike.setdefault((p.device, None if group["capturable"] else state["step"]), []).append(p)
            if group["capturable"] and alike:
                if len(alike) > 1:
                    raise ValueError("AdamW: with capturable, the parameters of a group are on one device")
                (device, _), = alike
                if "steps" not in group:
                    group["steps"] = torch.zeros((), dtype=torch.int64, device=device)
                group["steps"] += 1
            for (_, count), params in alike.items():
                states = [self.state[p] for p in params]
                ops.adamw_step(params, [p.grad for p in params], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states],
                               [s["scales"] for s in states] if group["bits"] == 8 else None, step=group["steps"] if group["capturable"] else count, lr=group["lr"],
                               betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], seed=group["seed"] + 0x1000193 * number)
        return loss

    def _check_capture(self):
        # what begins in a captured step would begin again at each replay, and a number that the host counts would stay where it is
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if params and not group["capturable"]:
                raise RuntimeError("AdamW: a step that is captured needs capturable=True")
            if params and ("steps" not in group or any(not self.state.get(p) for p in params)):
                raise RuntimeError("AdamW: the state begins in a step before the capture")

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # torch gives a state the type of its parameter; moments keep their own
        params = [p for group in self.param_groups for p in group["params"]]
        numbers = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(numbers, params):
            for name, value in state_dict["state"].get(i, {}).items():
                self.state[p][name] = value.detach().to(p.device, copy=True) if isinstance(value, torch.Tensor) else value
        for group in self.param_groups:
            if "steps" in group:
                group["steps"] = group["steps"].detach().to(group["params"][0].device, copy=True)
