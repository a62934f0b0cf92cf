"""Cross entropy over a vocabulary from hidden rows and output weights, without the logits."""
from __future__ import annotations

import torch

from ._train import native

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100, reduction: str = "mean") -> torch.Tensor:
    """``cross_entropy(x @ weight.T, targets)`` with gradients of ``x`` and ``weight``; the logits are formed in pieces and never stored.

    ``x`` (..., inner) and ``weight`` (vocabulary, inner): both bfloat16 or both float16, products and sums in float32; ``targets``: int64 of shape (...).
    Gives float32: a loss a row of shape (...) ("none"), their sum, or their mean over the rows that have a target (NaN if there are none).

    Rows whose target is ``ignore_index`` have a loss and a gradient of 0 whatever they hold, and enter that of ``weight`` times 0.  A target outside the vocabulary, and a row whose logits have a NaN or
    are infinite, gives NaN, in the gradients in its row of ``x`` and in all of ``weight``.

    The backward pass forms the logits again, a piece of the vocabulary at a time, and rounds their gradient to the operands' type for its products (float16 times a power of two
    that brings the largest of the rows' gradients into range).  It takes at most 384 MiB for a piece, or 1024 columns of it, beside float32 sums of the gradient of ``x`` (up to four of its size).
    Gradients have their tensors' types; all sums have a fixed order.

    Forward-mode derivatives, vmap and recorded (traced) calls raise NotImplementedError."""
    kind = REDUCTIONS.get(reduction)
    if kind is None:
        raise ValueError("linear_cross_entropy: reduction is one of %s" % ", ".join(REDUCTIONS))
    return native().linear_cross_entropy(x, weight, targets, ignore_index, kind)
