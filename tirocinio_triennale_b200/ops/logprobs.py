"""Log probabilities of given tokens, entropies and most likely tokens, with the gradient of the logits."""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ._train import TYPES, any_stride, call, floating, ptr, wants_grad

MOST_TOP = 64


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_tokens: torch.Tensor | None
    top_logprobs: torch.Tensor | None


def _forward(logits, tokens, top, ignore, keep):
    rows, vocab = logits.shape
    dev = logits.device
    both = torch.empty(2, rows, dtype=torch.float32, device=dev)
    logprobs, entropy = both.unbind(0)
    top_tokens = torch.empty(rows, top, dtype=torch.int64, device=dev) if top else None
    top_logprobs = torch.empty(rows, top, dtype=torch.float32, device=dev) if top else None
    stats = torch.empty(rows, 3, dtype=torch.float32, device=dev) if keep else None
    call("token_logprobs", "hc_token_logprobs", dev, logits.data_ptr(), TYPES[logits.dtype], rows, vocab, any_stride(logits),
         tokens.data_ptr(), ignore, top, logprobs.data_ptr(), entropy.data_ptr(), ptr(top_tokens), ptr(top_logprobs), ptr(stats))
    return logprobs, entropy, top_tokens, top_logprobs, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, ignore):
        logprobs, entropy, top_tokens, top_logprobs, stats = _forward(logits, tokens, top, ignore, True)
        ctx.save_for_backward(logits, tokens, stats)
        ctx.ignore = ignore
        if top:
            ctx.mark_non_differentiable(top_tokens, top_logprobs)
        ctx.set_materialize_grads(False)
        return logprobs, entropy, top_tokens, top_logprobs

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprobs, d_entropy, _tokens, _logprobs):
        logits, tokens, stats = ctx.saved_tensors
        if d_logprobs is None and d_entropy is None:
            return None, None, None, None
        rows, vocab = logits.shape
        d_logprobs = None if d_logprobs is None else d_logprobs.contiguous()
        d_entropy = None if d_entropy is None else d_entropy.contiguous()
        stride = any_stride(logits)
        # rows that begin at the same places of 16-byte groups as the logits', so that both move in whole groups; a product
        # whose rows were padded to such groups gets its gradient padded alike
        at = vocab + (stride - vocab) % 8
        d = torch.empty(rows * at, dtype=logits.dtype, device=logits.device).as_strided((rows, vocab), (at, 1))
        call("token_logprobs backward", "hc_token_logprobs_backward", logits.device, logits.data_ptr(), TYPES[logits.dtype], rows,
             vocab, stride, tokens.data_ptr(), ctx.ignore, stats.data_ptr(), ptr(d_logprobs), ptr(d_entropy), d.data_ptr(), at)
        return d, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of ``tokens`` under ``logits``, the entropy of every row, and its ``top`` most likely tokens.

    ``logits``: float32, bfloat16 or float16 of shape (..., vocabulary), rows any distance apart; ``tokens``: int64 of shape (...).
    Gives ``(logprobs, entropy, top_tokens, top_logprobs)``: the first two float32 of shape (...), both with a gradient for
    ``logits``; the last two of shape (..., top), the most likely token first and the lowest index first among equals, without
    gradient (None where ``top`` is 0; at most 64).  ``-logprobs.sum() / count`` is the cross-entropy loss.

    Rows whose token is ``ignore_index`` are not read: 0 for both numbers, -1 for their tokens, a gradient of 0.  Logits of -inf
    are tokens that cannot come: they add nothing and get a gradient of 0.  A row that has a NaN or +inf, or nothing above -inf,
    gives NaN and tokens of -1; a token outside the vocabulary gives NaN for its log probability and its row of the gradient."""
    floating("logits", logits)
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError("token_logprobs: logits have no vocabulary")
    vocab = logits.shape[-1]
    if vocab > 0x7FFFFFFF:
        raise ValueError("token_logprobs: a vocabulary of over 2^31 - 1 tokens")
    if not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int64 or tokens.device != logits.device:
        raise ValueError("token_logprobs: expected int64 tokens on the device of the logits")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError("token_logprobs: tokens of shape %s for logits of shape %s" % (tuple(tokens.shape), tuple(logits.shape)))
    top = int(top)
    if top < 0 or top > min(MOST_TOP, vocab):
        raise ValueError("token_logprobs: top is from 0 to %d" % min(MOST_TOP, vocab))
    shape = tokens.shape
    if logits.stride(-1) != 1 and vocab > 1:
        logits = logits.contiguous()
    flat = logits.reshape(-1, vocab)
    if flat.shape[0] > 1 and (flat.stride(0) < vocab or flat.stride(1) != 1):  # rows that overlap, as those of expand()
        flat = flat.contiguous()
    tokens = tokens.reshape(-1).contiguous()
    if wants_grad(flat):
        lp, ent, tt, tl = _TokenLogprobs.apply(flat, tokens, top, int(ignore_index))
    else:
        lp, ent, tt, tl, _ = _forward(flat, tokens, top, int(ignore_index), False)
    if len(shape) != 1:
        lp, ent = lp.reshape(shape), ent.reshape(shape)
        tt, tl = (None, None) if tt is None else (tt.reshape(*shape, top), tl.reshape(*shape, top))
    return TokenLogprobs(lp, ent, tt, tl)
