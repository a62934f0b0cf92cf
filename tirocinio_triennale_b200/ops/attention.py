"""Causal attention with a sliding window and first tokens that stay visible, and its backward pass."""
from __future__ import annotations

import torch

from ._train import native


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int | None = None, sinks: int = 0, scale: float | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` over what each query sees, with gradients of all three.

    ``q`` (batch, heads, queries, head size), ``k`` and ``v`` (batch, key heads, keys, head size): all bfloat16 or all float16; the head size a multiple of 8 up to 128; ``heads`` a
    multiple of the key heads, each of which as many query heads share, one after the other.  The queries are the last positions of the keys: query ``i`` stands at ``p = i + keys - queries`` (one
    query is a new token behind ``keys - 1`` others) and sees key ``j`` if ``j <= p`` and, with a ``window``, ``p - j < window`` or ``j < sinks``.  A query in front of the first key sees nothing and gives 0.
    ``scale``: above 0, 1 / sqrt(head size) unless given.

    The result has ``q``'s shape and lies as (batch, position, head, value), as a projection behind it reads it; so do the gradients.  Views whose values are adjacent, at
    16-byte boundaries and with strides of whole 16 bytes, are read where they lie, others are copied.  Scores, sums and statistics are float32; probabilities and their
    gradients are rounded to the operands' type before they enter products.  A key or value that is not finite may show in any query of its sequence and head, also in one that does not see it.

    Forward-mode derivatives, vmap and recorded (traced) calls raise NotImplementedError."""
    if window is not None and window < 1:
        raise ValueError("attention: a window is of at least one position")
    return native().attention(q, k, v, 0 if window is None else window, sinks, scale)
