"""Log probabilities of given tokens, entropies and most likely tokens, with the gradient of the logits."""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._train import native


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_tokens: torch.Tensor | None
    top_logprobs: torch.Tensor | None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of ``tokens`` under ``logits``, the entropy of every row, and its ``top`` most likely tokens.

    ``logits``: float32, bfloat16 or float16 of shape (..., vocabulary), rows any distance apart; ``tokens``: int64 of shape (...).
    Gives ``(logprobs, entropy, top_tokens, top_logprobs)``: the first two float32 of shape (...), both with a gradient for
    ``logits``; the last two of shape (..., top), the most likely token first and the lowest index first among equals, without
    gradient (None where ``top`` is 0; at most 64).  ``-logprobs.sum() / count`` is the cross-entropy loss.

    Rows whose token is ``ignore_index`` are not read: 0 for both numbers, -1 for their tokens, a gradient of 0.  Logits of -inf
    are tokens that cannot come: they add nothing and get a gradient of 0 (the row's own token: that of its log probability).  A row that has a NaN or +inf, or nothing above -inf,
    gives NaN and tokens of -1; a token outside the vocabulary gives NaN for its log probability and its row of the gradient.

    Forward-mode derivatives, vmap and recorded (traced) calls raise NotImplementedError."""
    return TokenLogprobs(*native().token_logprobs(logits, tokens, top, ignore_index))
