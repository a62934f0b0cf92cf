"""Layer norm with its backward pass on torch tensors."""
from __future__ import annotations

import torch

from ._train import native, type_code


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, with gradients of ``x``, ``weight`` and ``bias``.

    ``x``: float32, bfloat16 or float16, any shape; ``weight`` and ``bias``: one value per column, both of one of these types.
    The result has ``x``'s type, or ``out_dtype``: a float32 residual stream can give bfloat16 rows to a product, which saves a
    conversion.  Of the two 16-bit types one call takes only one.  Statistics and sums are held in float32; the sums of the
    gradients of ``weight`` and ``bias`` are formed in a fixed order.  Tensors with gaps are copied.

    Forward-mode derivatives, vmap and recorded (traced) calls raise NotImplementedError."""
    return native().layer_norm(x, weight, bias, eps, type_code(out_dtype))
