"""Newton-Schulz iteration of momentum matrices, as the Muon optimiser applies it."""
from __future__ import annotations

import torch

from ._train import native

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(update: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """``X = update / (|update| + eps)``, then ``steps`` times ``X = a X + (b S + c S S) X`` with ``S = X X^T``: the singular vectors
    stay, the singular values move to about 1.

    ``update``: float32, bfloat16 or float16 of shape (..., height, width); every matrix by itself, all of them in the same launches.
    The result is bfloat16 of the same shape.  Products take float16 operands and sum in float32, and X itself is carried to 22
    bits between the steps, so that directions that ``update`` hardly has gain nothing from rounding.  Coefficients
    with which the iteration may leave float16's range on its way raise ValueError (those in use stay far within it).  No gradient.

    Forward-mode derivatives, vmap and recorded (traced) calls raise NotImplementedError."""
    if len(coefficients) != 3:
        raise ValueError("orthogonalize: three coefficients")
    return native().orthogonalize(update, steps, *coefficients, eps)
