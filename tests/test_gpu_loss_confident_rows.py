"""Cross entropy from hidden rows where a row is sure of a token: what is left of the loss, and of the gradient at the token, is small beside the logits.

All rows of W are alike but for two of their values, so that logits differ by what these bring: `off` (a whole number) for a token that stands out, over a column of x that is 1, and nothing for the
column of x that is 0, which carries a token's mark into dx.  The loss is then log1p((vocabulary - 1) exp(-off)) at logits of any size, without rounding.

Tolerances.  u and h are half a step of fp32 and of the operands' type.  The sums of exponentials have their largest term, 1, and are off by u for each addition behind it: 16 and 5 in a
stretch of columns, 31 and 32 where stretches are joined, twice that for products with powers of two that are 1 only to a step; the others are off by 4 u + 3 u off of themselves.  The sums
that logits are differ in their last step alone: by 4 whole steps of fp32 at the logit's size, for the instruction's addition and that of a part of the sum."""
import math

import pytest
import torch

from tirocinio_triennale_b200 import ops

U = torch.finfo(torch.float32).eps / 2
BF16, F16 = torch.bfloat16, torch.float16
ADDITIONS = 2 * (16 + 5 + 31 + 32)


def make(rows, inner, vocab, size, off, kind, stands_out, exact=False, seed=0):
    """x and W of logits of about `size`; of each row token `stands_out` is `off` above the others."""
    g = torch.Generator().manual_seed(seed + rows + inner)
    x, w = torch.zeros(rows, inner), torch.zeros(vocab, inner)
    if exact:  # one product of powers of two, the same in all rows
        x[:, 0], w[:, 0] = 2.0 ** 4, size / 2.0 ** 4
    else:  # sums of products that are all positive
        x[:, :inner - 2] = 0.5 + torch.rand(rows, inner - 2, generator=g)
        w[:, :inner - 2] = (0.5 + torch.rand(inner - 2, generator=g)) * size / inner
    x[:, -1] = 1.0
    w[:, -1] = -off
    w[stands_out, -1] = 0.0
    w[stands_out, -2] = 1.0  # where x is 0: dx there is G of that token
    return x.to(kind).cuda(), w.to(kind).cuda()


def room_of(loss, logit, off):
    """of a loss, relative to itself"""
    return U * ADDITIONS / loss + U * (8 + 3 * off) + 4 * 2 * U * 2.0 ** math.ceil(math.log2(logit))


SIZES = [(1, 64, 16), (5, 3, 7), (16, 1000, 1000), (17, 40, 64), (300, 700, 100), (700, 3001, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("size", [16, 512, 8192])
@pytest.mark.parametrize("rows,vocab,inner", SIZES)
def test_small_losses_beside_large_logits(rows, vocab, inner, size, kind):
    for off in (4, 9, 13):
        x, w = make(rows, inner, vocab, size, off, kind, vocab // 2, exact=True)
        t = torch.full((rows,), vocab // 2, device="cuda")
        want = math.log1p((vocab - 1) * math.exp(-off))
        room = want * room_of(want, size, off) - want * 8 * U * 2.0 ** math.ceil(math.log2(size))  # these sums are exact
        for reduction in ("none", "mean", "sum"):
            loss = ops.linear_cross_entropy(x, w, t, reduction=reduction).double() / (rows if reduction == "sum" else 1)
            assert ((loss - want).abs() <= 1.01 * room + U * want).all(), (float((loss - want).abs().max()), want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("rows,vocab,inner", SIZES + [(16, 50257, 64), (33, 13001, 16)])
def test_losses_far_below_one(rows, vocab, inner, kind):
    """Their digits are those of the others' sum, in which the token's own 1 has no part."""
    for size in (16, 8192):
        for off in (16, 24, 32):
            x, w = make(rows, inner, vocab, size, off, kind, vocab - 1, exact=True)
            want = math.log1p((vocab - 1) * math.exp(-off))
            loss = ops.linear_cross_entropy(x, w, torch.full((rows,), vocab - 1, device="cuda"), reduction="none").double()
            assert ((loss - want).abs() <= want * U * (ADDITIONS + 8 + 3 * off)).all(), (float((loss - want).abs().max()), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 40])
def test_logits_that_are_no_numbers(rows):
    """Of the token itself, or of another one."""
    inner, vocab = 8, 700
    for token in (3, 699):
        for at in (3, 699):
            for value, want in ((math.inf, math.nan), (math.nan, math.nan), (-math.inf, math.inf if at == token else math.log(vocab - 1))):
                w = torch.zeros(vocab, inner, dtype=BF16, device="cuda")
                x = torch.ones(rows, inner, dtype=BF16, device="cuda")
                w[at, 0] = value
                loss = ops.linear_cross_entropy(x, w, torch.full((rows,), token, device="cuda"), reduction="none")
                assert torch.allclose(loss, torch.full_like(loss, want), rtol=1e-5, atol=0, equal_nan=True), (token, at, value)
        w = torch.full((vocab, inner), -math.inf, dtype=BF16, device="cuda")
        t = torch.full((rows,), token, device="cuda")
        assert ops.linear_cross_entropy(x, w, t, reduction="none").isnan().all()
        w[token] = 1.0  # and no other
        assert (ops.linear_cross_entropy(x, w, t, reduction="none") == 0).all()
    assert (ops.linear_cross_entropy(x, w[token:token + 1], torch.zeros_like(t), reduction="none") == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 16, 17, 300])
@pytest.mark.parametrize("inner,size", [(64, 20), (768, 20), (768, 400), (2048, 20), (4096, 20), (4096, 400)])
def test_gradients_of_small_losses(inner, size, rows, kind):
    """G at the token is -(1 - p), whatever the logits' size: dx at the token's mark, and the token's row of dW."""
    h, vocab, off = torch.finfo(kind).eps / 2, 67, 13
    x, w = make(rows, inner, vocab, size, off, kind, 5)
    t = torch.full((rows,), 5, device="cuda")
    rest = (vocab - 1) * math.exp(-off)
    want = rest / (1 + rest)
    logit = (x.double() @ w.double()[5]).max().item()
    for reduction, a in (("none", None), ("sum", 1.0), ("mean", 64.0)):
        leaves = [v.detach().requires_grad_() for v in (x, w)]
        got = ops.linear_cross_entropy(*leaves, t, reduction=reduction)
        weights = torch.linspace(0.5, 2.0, rows, device="cuda") if reduction == "none" else torch.full((rows,), a / (rows if reduction == "mean" else 1), device="cuda")
        dx, dw = torch.autograd.grad(got, leaves, weights if reduction == "none" else torch.tensor(a, device="cuda"))
        G = -weights.double() * want
        # the loss, of which the others' sum is off relative to itself; G, rounded
        room = U * (ADDITIONS + 12 + 3 * off) + 4 * 2 * U * 2.0 ** math.ceil(math.log2(2 * logit)) + h + 4 * U
        least = 2.0 ** -24 if kind == F16 else 0.0  # dx and dW have no smaller steps; those of G are 2^-37 of the largest weight
        lost = 2.0 ** -37 * weights.double().max() if kind == F16 else 0.0
        assert ((dx[:, -2].double() - G).abs() <= 1.01 * ((room + h) * G.abs() + lost + least)).all(), float(((dx[:, -2].double() - G) / G).abs().max())
        exact = G @ x.double()
        size_of = G.abs() @ x.double().abs()
        assert ((dw[5].double() - exact).abs() <= 1.01 * ((room + (rows / 16 + 20) * 2 * U) * size_of + h * exact.abs() + lost * x.double().abs().sum(0) + least)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 16, 17, 300])
@pytest.mark.parametrize("inner", [1024, 1025, 4096, 8192, 16384])
def test_probabilities_belong_to_the_sums(inner, rows, kind):
    """A token that a row is sure of, and that is not its own: its p is 1, with logits that are long sums of one sign.  Both passes take them from sums of the same parts, so that what the tensor core
    loses of each, 6.5e-9 of it a term within a part of 1024, is lost in both: what they may differ by is that of one part, where few rows' sums go through another instruction."""
    h, vocab, off, size = torch.finfo(kind).eps / 2, 67, 40, 900
    x, w = make(rows, inner, vocab, size, off, kind, 5)
    t = torch.full((rows,), 6, device="cuda")
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    dx, _ = torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, reduction="sum"), leaves)
    logit = (x.double() @ w.double()[5]).max().item()
    room = 2 * h + 8 * U + 4 * 2 * U * 2.0 ** math.ceil(math.log2(logit)) + (6.5e-9 * 1024 * logit if rows <= 16 else 0.0)
    assert ((dx[:, -2].double() - 1).abs() <= 1.01 * room).all(), float((dx[:, -2].double() - 1).abs().max())
