"""One AdamW step over many tensors, with moments in 32 or in 8 bits."""
from __future__ import annotations

import torch

from ._train import native

BLOCK = 256  # values that share their scales


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales=None, *, step: int | torch.Tensor, lr: float | torch.Tensor = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.01, seed: int = 0) -> None:
    """``m = b1 m + (1 - b1) g``, ``v = b2 v + (1 - b2) g^2``,
    ``p = p (1 - lr weight_decay) - m / (sqrt(v) / sqrt(1 - b2^step) + eps) lr / (1 - b1^step)``, in place, for all tensors of the lists in one launch.

    ``params``: float32, bfloat16 or float16 CUDA tensors of one device without gaps, any sizes; ``grads``: of the same shapes, of the
    parameter's type or, for float32 parameters, any of the three.  All arithmetic is float32; a 16-bit parameter is rounded once.

    Without ``scales`` the moments ``exp_avgs`` and ``exp_avg_sqs`` are float32, with the shapes and strides of the parameters.  With ``scales`` they are uint8:
    ``m`` as sign, 4 bits of exponent and 3 of fraction, ``sqrt(v)`` as 4 and 4 bits, relative to the largest of each 256 values (in the
    order of memory), which ``scales`` (float32, two columns, a row for every 256 values) has.  Zeros everywhere are the state to begin with.
    Both are rounded up or down at random in proportion to what is lost, so that they follow the averages although a step moves them by less than their
    last bit; the random bits are a function of the value's place, the tensor's place in the list, ``step`` and ``seed``, and the same
    call gives the same bits.  A block of 256 whose moments are no longer finite becomes NaN as a whole.

    ``step``, the number of this step, from 1, and ``lr`` may be CUDA tensors of one value (int64, float32): a captured call then goes on counting.
    Tensors that overlap, or the same one twice, raise ValueError."""
    step_at, lr_at = (step if isinstance(step, torch.Tensor) else None), (lr if isinstance(lr, torch.Tensor) else None)
    native().adamw_step(params, grads, exp_avgs, exp_avg_sqs, scales, 0.0 if lr_at is not None else lr, lr_at, betas[0], betas[1], eps, weight_decay,
                        0 if step_at is not None else step, step_at, seed & 0xFFFFFFFFFFFFFFFF)


def adamw_values(exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, scales: torch.Tensor):
    """What moments in 8 bits stand for: ``m`` and ``v`` in float32, of the shape of ``exp_avg`` (uint8, whole blocks of 256 from its first value on)."""
    return native().adamw_values(exp_avg, exp_avg_sq, scales)
