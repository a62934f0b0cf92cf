"""Newton-Schulz iteration of momentum matrices, as the Muon optimiser applies it."""
from __future__ import annotations

import torch

from ._train import TYPES, call, floating, size

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def orthogonalize(update: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """``X = update / (|update| + eps)``, then ``steps`` times ``X = a X + (b S + c S S) X`` with ``S = X X^T``: the singular vectors
    stay, the singular values move to about 1.

    ``update``: float32, bfloat16 or float16 of shape (..., height, width); every matrix by itself, all of them in the same launches.
    The result is bfloat16 of the same shape.  Products take float16 operands and sum in float32, and X itself is carried to 22
    bits between the steps, so that directions that ``update`` hardly has gain nothing from rounding.  No gradient."""
    floating("update", update)
    if update.dim() < 2 or 0 in update.shape[-2:]:
        raise ValueError("orthogonalize: expected matrices, got shape %s" % (tuple(update.shape),))
    if not 1 <= int(steps) <= 100 or len(coefficients) != 3 or not eps >= 0:
        raise ValueError("orthogonalize: 1 to 100 steps, three coefficients, eps not negative")
    height, width = update.shape[-2:]
    flat = update.detach().reshape(-1, height, width)
    if (flat.stride(2) != 1 and width > 1) or (height > 1 and flat.stride(1) < width):
        flat = flat.contiguous()
    batch = flat.shape[0]
    if batch > 65535 or max(height, width) >= 1 << 24:
        raise ValueError("orthogonalize: at most 65535 matrices with sides below 2^24")
    dev = update.device
    out = torch.empty(update.shape, dtype=torch.bfloat16, device=dev)
    need = size("hc_orthogonalize_bytes", dev, batch, height, width)
    scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    call("orthogonalize", "hc_orthogonalize", dev, flat.data_ptr(), TYPES[flat.dtype], batch, height, width,
         flat.stride(1) if height > 1 else width, flat.stride(0) if batch > 1 else 0, out.data_ptr(), int(steps), *map(float, coefficients),
         float(eps), None if scratch is None else scratch.data_ptr(), need)
    return out
