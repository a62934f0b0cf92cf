"""Matrix product with bias, activation and residual in its epilogue, and its backward pass."""
from __future__ import annotations

import torch

from ._train import native, type_code

ACTIVATIONS = {None: 0, "gelu_tanh": 1, "relu": 2, "silu": 3}


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
           residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` with gradients of all four tensors.

    ``x`` (..., inner) and ``weight`` (width, inner): both bfloat16 or both float16, products summed in float32.  ``bias``: one value
    per column, of any of the three types.  ``activation``: None, "gelu_tanh", "relu" or "silu".  ``residual``: of the result's shape,
    float32 or ``x``'s type, and the result has its type; without one the result has ``x``'s type or ``out_dtype`` (float32).

    Everything behind the product happens before the result is stored.  For the backward pass of an activation its argument is
    kept in ``x``'s type, and the gradient is rounded to that type before it enters the products (a float32 one, where that
    type is float16, times a power of two that brings its largest value into range); gradients of ``x`` and ``weight``
    have their types, that of ``bias`` its own, summed in float32 in a fixed order.  Where eight does not divide ``width`` the
    result's rows are kept apart so that they begin at 16-byte boundaries: it has gaps.

    Forward-mode derivatives, vmap and recorded (traced) calls raise NotImplementedError."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError("linear: activation is one of %s" % ", ".join(map(str, ACTIVATIONS)))
    return native().linear(x, weight, bias, act, residual, type_code(out_dtype))
