"""Log probabilities, entropies, most likely tokens and the gradient of logits against the formulas in 64 bits.

Tolerances count roundings; u is half a step of fp32.  A thread adds at most vocabulary / 512 + 8 terms in a line, some 16
more join the threads; exp of a difference d is off by |d| u * 2.5 for its argument and 2 u for the function itself, and
exp(d) |d| stays below 0.4.  With n = vocabulary / 512 + 48 the log of the sum is off by at most n u, as are the sums around
it in units of their absolute terms."""
import ctypes as C
import math

import pytest
import torch

from tirocinio_triennale_b200 import _lib, ops

U = torch.finfo(torch.float32).eps / 2
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
IGNORED = -100


def make(rows, vocab, kind, seed, masked=False, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    t = torch.randint(0, vocab, (rows,), generator=g)
    if masked:
        x[torch.rand(rows, vocab, generator=g) < 0.4] = -math.inf
        x[torch.arange(rows), t] = 1.0
    if rows > 4:
        t[3] = IGNORED
    return x.to(kind).cuda(), t.cuda(), torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()


def check(x, t, a, b, top=0):
    vocab = x.shape[1]
    n = vocab / 512 + 48
    leaf = x.detach().requires_grad_()
    r = ops.token_logprobs(leaf, t, top=top)
    (dx,) = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (a, b))
    plain = ops.token_logprobs(x, t, top=top)
    for p, q in zip(r, plain):
        assert p is q is None or torch.equal(p, q)
    X, kept = x.double(), t != IGNORED
    at = torch.where(kept, t, 0)[:, None]
    m = X.max(1, keepdim=True).values
    log_s = torch.logsumexp(X - m, 1, keepdim=True)
    logp = X - m - log_s
    p = logp.exp()
    pl = torch.where(p > 0, p * logp, 0.0)
    h = -pl.sum(1)
    want = torch.where(kept, logp.gather(1, at)[:, 0], 0.0)
    room = 1.01 * U * (n + 3 * (logp.gather(1, at)[:, 0].abs() + log_s[:, 0]))
    assert ((r.logprobs.double() - want).abs() <= room).all()
    spread = (p * torch.where(p > 0, X - m, 0.0).abs()).sum(1)
    assert ((r.entropy.double() - torch.where(kept, h, 0.0)).abs() <= 1.01 * U * (n + (2 * n + 8) * (1 + spread) + 3 * log_s[:, 0])).all()
    A, B = (v.double()[:, None] * kept[:, None] for v in (a, b))
    want = -A * p - B * torch.where(p > 0, p * (logp + h[:, None]), 0.0)
    want.scatter_add_(1, at, A)
    off = U * (2 * n + 12 + 6 * torch.where(p > 0, logp, 0.0).abs())  # of p, relative
    size = p * (A.abs() + B.abs() * (torch.where(p > 0, logp, 0.0).abs() + h.abs()[:, None] + 1 + spread[:, None]))
    step = torch.finfo(x.dtype).eps / 2
    tol = step * want.abs() + 1.05 * off * size + U * A.abs() + (2.0 ** -25 if x.dtype == F16 else 1e-37)
    assert ((dx.double() - want).abs() <= tol).all()
    assert not dx[~kept].any() and dx.shape == x.shape and dx.dtype == x.dtype
    if top:
        value, i = torch.sort(x, dim=1, descending=True, stable=True)
        assert torch.equal(r.top_tokens, torch.where(kept[:, None], i[:, :top], -1))
        lp = (value[:, :top].double() - m - log_s)
        lp = torch.where(kept[:, None], lp, 0.0)
        same = (r.top_logprobs.double() == lp) | ((r.top_logprobs.double() - lp).abs() <= 1.01 * U * (n + 3 * (lp.abs() + log_s)))
        assert same.all()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 63, 257, 1000, 4095, 4096, 4097, 8193, 32000, 50257, 131071])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_vocabularies(vocab, kind):
    x, t, a, b = make(9, vocab, kind, vocab)
    check(x, t, a, b, min(5, vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 36, 37, 73, 74, 75, 147, 149, 1500])
@pytest.mark.parametrize("vocab", [2049, 50257])
def test_rows(rows, vocab):
    x, t, a, b = make(rows, vocab, BF16, rows)
    check(x, t, a, b, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [1, 2, 15, 16, 17, 20, 33, 64])
@pytest.mark.parametrize("rows,vocab", [(1, 50257), (3, 64), (5, 300), (40, 4100), (200, 9001)])
def test_top(top, rows, vocab):
    x, t, a, b = make(rows, vocab, BF16, top)
    check(x, t, a, b, top)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_masked_logits(rows, kind):
    x, t, a, b = make(rows, 5000, kind, 1, masked=True)
    check(x, t, a, b, 20)
    x[:, 7:] = -math.inf  # fewer tokens than asked for: those that cannot come follow, lowest first
    x[:, :7] = torch.arange(7, device="cuda").to(kind)
    t = torch.where(t == IGNORED, t, t % 7)
    check(x, t, a, b, 20)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_masks_of_the_lowest_value(kind):
    x, t, a, b = make(6, 700, kind, 2)
    low = torch.finfo(kind).min
    x[0] = low
    x[1, 1:] = low
    x[2, :350] = low
    t[1], t[2] = 0, 600
    check(x, t, a, b, 4)
    x = torch.full((2, 600), low, dtype=kind, device="cuda")
    x[1, 599] = torch.finfo(kind).max
    r = ops.token_logprobs(x, torch.tensor([5, 599], device="cuda"), top=2)
    assert abs(float(r.logprobs[0]) + math.log(600)) < 1e-5 and float(r.logprobs[1]) == 0 and float(r.entropy[1]) == 0
    assert r.top_tokens.tolist() == [[0, 1], [599, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 50257])
def test_equal_logits_and_zeros_of_both_signs(vocab):
    x = torch.zeros(3, vocab, device="cuda")
    x[1, ::2] = -0.0
    x[2] = 3.5
    t = torch.tensor([0, 1, vocab - 1], device="cuda")
    one = torch.ones(3, device="cuda")
    check(x, t, one, one, 32)


@pytest.mark.gpu
def test_largest_logits_at_one_thread():
    """The groups of a thread are 512 groups apart: with the largest logits all there, its share outgrows the candidates' list."""
    vocab = 262144 * 4
    x = torch.zeros(2, vocab, device="cuda")
    g = torch.Generator().manual_seed(3)
    for thread in range(40):
        at = (torch.arange(thread * 8, vocab, 4096)[:, None] + torch.arange(8)).reshape(-1)
        x[:, at.cuda()] = 5 + torch.rand(2, at.numel(), generator=g).cuda()
    t = torch.tensor([1, 2], device="cuda")
    one = torch.ones(2, device="cuda")
    check(x, t, one, one, 64)
    check(x.repeat(40, 1), t.repeat(40), one.repeat(40), one.repeat(40), 64)


@pytest.mark.gpu
def test_rows_without_a_distribution():
    x, t, a, b = make(8, 1000, F32, 4)
    x[0] = -math.inf
    x[1, 5] = math.nan
    x[2, 5] = math.inf
    t[4] = 1000
    t[5] = -1
    leaf = x.detach().requires_grad_()
    r = ops.token_logprobs(leaf, t, top=3)
    (dx,) = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (a, b))
    assert torch.isnan(r.logprobs[[0, 1, 2, 4, 5]]).all() and torch.isnan(r.entropy[:3]).all() and torch.isfinite(r.entropy[3:]).all()
    assert (r.top_tokens[:3] == -1).all() and torch.isnan(r.top_logprobs[:3]).all() and (r.top_tokens[3] == -1).all()
    assert torch.isnan(dx[[0, 1, 2, 4, 5]]).all() and torch.isfinite(dx[[3, 6, 7]]).all()
    x[3] = math.nan  # a row that is left out may hold anything
    r = ops.token_logprobs(x, t)
    assert float(r.logprobs[3]) == 0 and float(r.entropy[3]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 3, 7, 8, 100])
def test_rows_apart(pad):
    g = torch.Generator().manual_seed(pad)
    wide = torch.randn(20, 777 + pad, generator=g).to(BF16).cuda()
    t = torch.randint(0, 777, (20,), generator=g).cuda()
    a, b = torch.randn(20, generator=g).cuda(), torch.randn(20, generator=g).cuda()
    check(wide[:, :777], t, a, b, 3)
    check(wide[:, pad:], t, a, b, 3)
    check(wide.t().contiguous().t()[:, :777], t, a, b, 3)
    check(wide[:1, :777].expand(20, 777), t, a, b, 3)


@pytest.mark.gpu
def test_shapes_and_single_gradients():
    x, t, a, b = make(12, 333, BF16, 5)
    whole = ops.token_logprobs(x, t, top=2)
    shaped = ops.token_logprobs(x.view(3, 4, 333), t.view(3, 4), top=2)
    assert shaped.logprobs.shape == (3, 4) and shaped.top_tokens.shape == (3, 4, 2)
    assert all(torch.equal(p.flatten(), q.flatten()) for p, q in zip(whole, shaped))
    one = ops.token_logprobs(x[0], t[0])
    assert one.logprobs.shape == () and one.logprobs == whole.logprobs[0] and one.top_tokens is None
    leaf = x.detach().requires_grad_()
    r = ops.token_logprobs(leaf, t)
    (d,) = torch.autograd.grad(-r.logprobs.sum() / 11, (leaf,))  # the trainer's loss: a gradient with strides of 0
    want = torch.nn.functional.cross_entropy(leaf.double(), t, ignore_index=IGNORED)
    (w,) = torch.autograd.grad(want, (leaf,))
    assert ((d.double() - w.double()).abs() <= 2 ** -7 * w.double().abs() + 2.0 ** -20).all()  # both are rounded to bf16
    r = ops.token_logprobs(leaf, t)
    (d,) = torch.autograd.grad(r.entropy.sum(), (leaf,))
    assert torch.isfinite(d).all()
    empty = ops.token_logprobs(x[:0], t[:0], top=2)
    assert empty.logprobs.shape == (0,) and empty.top_tokens.shape == (0, 2)


@pytest.mark.gpu
def test_same_bits_every_time_other_streams_and_graphs():
    x, t, a, b = make(64, 50257, BF16, 6)

    def step():
        leaf = x.detach().requires_grad_()
        r = ops.token_logprobs(leaf, t, top=8)
        return (*r, *torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (a, b)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = step()
    x.copy_(x.flip(0))
    other = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, there))
    assert all(torch.equal(p, q) for p, q in zip(other, caught))


@pytest.mark.gpu
def test_refusals():
    x, t = torch.randn(4, 16, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in (lambda: ops.token_logprobs(x.double(), t), lambda: ops.token_logprobs(x, t.int()), lambda: ops.token_logprobs(x, t[:3]),
                lambda: ops.token_logprobs(x, t.cpu()), lambda: ops.token_logprobs(x, t, top=17), lambda: ops.token_logprobs(x, t, top=-1),
                lambda: ops.token_logprobs(x[:, :0], t), lambda: ops.token_logprobs(x.repeat(1, 8), t, top=65)):
        with pytest.raises(ValueError):
            bad()


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        ops.token_logprobs(torch.ones(2, 8), torch.zeros(2, dtype=torch.int64))
    lib = _lib.cuda()
    p = C.c_void_p(4096)  # never read: every call below is refused before anything is launched
    good = dict(x=p, type=1, rows=4, vocab=16, stride=16, tokens=p, ignore=-100, top=2, lp=p, h=p, tt=p, tl=p, st=None)

    def forward(**kw):
        return lib.hc_token_logprobs(*{**good, **kw}.values(), None)

    for kw in (dict(type=3), dict(vocab=0), dict(vocab=1 << 31, stride=1 << 31), dict(stride=15), dict(top=65), dict(top=-1), dict(top=17), dict(x=None),
               dict(x=C.c_void_p(4097)), dict(tokens=None), dict(lp=None), dict(h=None), dict(tt=None), dict(tl=None), dict(rows=1 << 50)):
        assert forward(**kw) == 4, kw
    assert forward(rows=0) == 0
    back = lambda **kw: lib.hc_token_logprobs_backward(*{**dict(x=p, type=1, rows=4, vocab=16, stride=16, tokens=p, ignore=-100, st=p, a=p, b=p, dx=p, ds=16), **kw}.values(), None)  # noqa: E731
    for kw in (dict(st=None), dict(tokens=None), dict(dx=None), dict(ds=15), dict(type=5)):
        assert back(**kw) == 4, kw
    assert back(rows=0) == 0


# From 1184 rows and a vocabulary of 8192 up, blocks stay and rows stream through them.
@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [8192, 8193, 12301])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("top", [0, 20])
@pytest.mark.parametrize("masked", [False, True])
def test_many_rows(vocab, kind, top, masked):
    x, t, a, b = make(1200, vocab, kind, vocab, masked)
    t[700:1190] = IGNORED  # blocks that skip rows, some at their first one
    check(x, t, a, b, top)


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 3, 8, 102])
def test_many_rows_apart(pad):
    g = torch.Generator().manual_seed(pad)
    wide = torch.randn(2500, 8197 + pad, generator=g).to(BF16).cuda()
    t = torch.randint(0, 8197, (2500,), generator=g).cuda()
    a, b = torch.randn(2500, generator=g).cuda(), torch.randn(2500, generator=g).cuda()
    check(wide[:, :8197], t, a, b, 3)
    check(wide[:, pad:], t, a, b, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_many_rows_of_which_some_have_no_distribution(kind):
    x, t, a, b = make(1300, 8201, kind, 5)
    want = ops.token_logprobs(x, t, top=4)
    bad = {0: math.nan, 7: math.inf, 650: math.nan, 1299: -math.inf}
    x[0, 0], x[7, 8200], x[650, 4000], x[1299] = math.nan, math.inf, math.nan, -math.inf
    low = torch.finfo(kind).min
    x[20], x[21, 1:] = low, low
    t[20], t[21] = 3, 0
    leaf = x.detach().requires_grad_()
    r = ops.token_logprobs(leaf, t, top=4)
    (dx,) = torch.autograd.grad((r.logprobs, r.entropy), (leaf,), (a, b))
    rows = list(bad)
    assert torch.isnan(r.logprobs[rows]).all() and torch.isnan(r.entropy[rows]).all() and (r.top_tokens[rows] == -1).all() and torch.isnan(dx[rows]).all()
    keep = [i for i in range(1300) if i not in bad and i not in (20, 21)]
    for p, q in zip(r, want):
        assert torch.equal(p[keep], q[keep])
    check(x[[i for i in range(1300) if i not in bad]], t[[i for i in range(1300) if i not in bad]], a[:1296], b[:1296], 4)


@pytest.mark.gpu
def test_largest_logits_at_one_thread_of_many_rows():
    """The same where rows stream: the groups of a thread are 128 groups apart, and 40 of the threads have all that counts."""
    vocab = 65536
    x = torch.zeros(1190, vocab, device="cuda")
    g = torch.Generator().manual_seed(3)
    for thread in range(40):
        at = (torch.arange(thread * 8, vocab, 1024)[:, None] + torch.arange(8)).reshape(-1)
        x[:, at.cuda()] = 5 + torch.rand(1190, at.numel(), generator=g).cuda()
    t = torch.arange(1190, device="cuda")
    one = torch.ones(1190, device="cuda")
    check(x, t, one, one, 64)
