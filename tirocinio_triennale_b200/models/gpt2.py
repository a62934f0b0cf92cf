"""GPT-2-shaped decoder (12 layers, d_model 768, 12 heads, vocab 50257 for "small") used by the
data-parallel benchmark: random-init weights, uniform random token ids.  Plain PyTorch modules
(bf16 autocast, fused scaled-dot-product attention); the point of the benchmark is the gradient
allreduce, which is this library's compressed collective.

With ``GPT2Config.fused`` the same weights run through this library's operators on a CUDA device:
the residual stream stays float32, norms give bfloat16 rows to the products, bias, GELU and residual
are added where a product is stored, and the loss takes one pass over the logits and one for their
gradient (``ops.layer_norm``, ``ops.linear``, ``ops.token_logprobs``).  No autocast is needed."""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


@dataclass
class GPT2Config:
    n_layer: int = 12
    n_head: int = 12
    d_model: int = 768
    vocab_size: int = 50257
    seq_len: int = 1024
    dropout: float = 0.0
    fused: bool = False  # this library's operators in place of torch's (CUDA, float32 weights, bfloat16 products)

    @staticmethod
    def small():
        return GPT2Config()

    @staticmethod
    def tiny():
        return GPT2Config(n_layer=2, n_head=2, d_model=64, vocab_size=257, seq_len=32)


def _norm(x, m: nn.LayerNorm):
    return ops.layer_norm(x, m.weight, m.bias, eps=m.eps, out_dtype=torch.bfloat16)


def _linear(x, m: nn.Linear, **kw):
    return ops.linear(x, m.weight.to(torch.bfloat16), m.bias, **kw)


class Block(nn.Module):
    def __init__(self, cfg: GPT2Config):
        super().__init__()
        self.ln1 = nn.LayerNorm(cfg.d_model)
        self.qkv = nn.Linear(cfg.d_model, 3 * cfg.d_model)
        self.proj = nn.Linear(cfg.d_model, cfg.d_model)
        self.ln2 = nn.LayerNorm(cfg.d_model)
        self.fc = nn.Linear(cfg.d_model, 4 * cfg.d_model)
        self.out = nn.Linear(4 * cfg.d_model, cfg.d_model)
        self.n_head = cfg.n_head
        self.fused = cfg.fused

    def forward(self, x):
        B, T, C = x.shape
        q, k, v = (_linear(_norm(x, self.ln1), self.qkv) if self.fused else self.qkv(self.ln1(x))).split(C, dim=2)
        q = q.view(B, T, self.n_head, C // self.n_head).transpose(1, 2)
        k = k.view(B, T, self.n_head, C // self.n_head).transpose(1, 2)
        v = v.view(B, T, self.n_head, C // self.n_head).transpose(1, 2)
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        if self.fused:
            x = _linear(a.transpose(1, 2).reshape(B, T, C), self.proj, residual=x)
            return _linear(_linear(_norm(x, self.ln2), self.fc, activation="gelu_tanh"), self.out, residual=x)
        x = x + self.proj(a.transpose(1, 2).reshape(B, T, C))
        return x + self.out(F.gelu(self.fc(self.ln2(x)), approximate="tanh"))


class GPT2(nn.Module):
    def __init__(self, cfg: GPT2Config):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab_size, cfg.d_model)
        self.wpe = nn.Embedding(cfg.seq_len, cfg.d_model)
        self.blocks = nn.ModuleList([Block(cfg) for _ in range(cfg.n_layer)])
        self.ln_f = nn.LayerNorm(cfg.d_model)
        self.apply(self._init)
        for b in self.blocks:  # GPT-2's scaled init of the residual projections
            for w in (b.proj.weight, b.out.weight):
                nn.init.normal_(w, 0.0, 0.02 / math.sqrt(2 * cfg.n_layer))

    @staticmethod
    def _init(m):
        if isinstance(m, (nn.Linear, nn.Embedding)):
            nn.init.normal_(m.weight, 0.0, 0.02)
        if isinstance(m, nn.Linear) and m.bias is not None:
            nn.init.zeros_(m.bias)

    def forward(self, idx, targets=None):
        B, T = idx.shape
        pos = torch.arange(T, device=idx.device)
        x = self.wte(idx) + self.wpe(pos)
        for b in self.blocks:
            x = b(x)
        if self.cfg.fused:
            logits = ops.linear(_norm(x, self.ln_f), self.wte.weight.to(torch.bfloat16))
            if targets is None:
                return logits
            kept = (targets != -100).sum()  # as cross_entropy leaves rows out
            return -ops.token_logprobs(logits, targets).logprobs.sum() / kept
        logits = F.linear(self.ln_f(x), self.wte.weight)  # tied output embedding
        if targets is None:
            return logits
        return F.cross_entropy(logits.float().view(-1, logits.size(-1)), targets.reshape(-1))
