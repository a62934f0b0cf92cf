"""Cross entropy from hidden rows and output weights, and its gradients, against the formulas in 64 bits.

Tolerances count roundings.  u and h are half a step of fp32 and of the operands' type.  A logit is a sum over k products, which are exact in fp32, through at most k / 16 + 20 additions in a
line, each off by at most a whole step (the tensor core need not round to nearest): off by e.  An exponential is off by 4 u for the function, and by its argument's error
(at most e twice, and 3 u of the argument); a sum of exponentials goes through at most 16 + 4 additions of a stretch, vocabulary / 1024 + 64 of the stretches' and as many products with
powers of two.  G is rounded once to the operands' type; its products are sums like those of the logits, over the vocabulary and its pieces or over the rows."""
import ctypes as C
import math

import pytest
import torch

from tirocinio_triennale_b200 import _lib, ops
from tirocinio_triennale_b200.models import GPT2, GPT2Config

U = torch.finfo(torch.float32).eps / 2
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
IGNORED = -100


def sums(k):
    return (k / 16 + 20) * 2 * U


def make(rows, inner, vocab, kind, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, inner, generator=g)
    w = torch.randn(vocab, inner, generator=g) * (scale / inner ** 0.5)
    t = torch.randint(0, vocab, (rows,), generator=g)
    x[::2] += 2 * w[t[::2]]  # rows that know their token
    if rows > 4:
        t[3] = IGNORED
    return x.to(kind).cuda(), w.to(kind).cuda(), t.cuda(), torch.randn(rows, generator=g).cuda()


def check(x, w, t, a, reduction="none", upstream=1.0):
    h, least = torch.finfo(x.dtype).eps / 2, 2.0 ** -25 if x.dtype == F16 else 1e-37
    rows, (vocab, inner) = x.numel() // x.shape[-1], w.shape
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    loss = ops.linear_cross_entropy(*leaves, t, reduction=reduction)
    assert loss.dtype == F32 and loss.shape == (t.shape if reduction == "none" else ())
    assert torch.equal(loss, ops.linear_cross_entropy(x, w, t, reduction=reduction))
    given = a.view(t.shape) if reduction == "none" else torch.tensor(upstream, device="cuda")
    dx, dw = torch.autograd.grad(loss, leaves, given, retain_graph=True)
    assert dx.shape == x.shape and dx.dtype == x.dtype and dw.shape == w.shape and dw.dtype == w.dtype
    for i in (0, 1):  # one alone
        assert torch.equal(torch.autograd.grad(loss, leaves[i], given, retain_graph=True)[0], (dx, dw)[i])
    X, W, T = x.double().reshape(rows, inner), w.double(), t.reshape(-1)
    kept = T != IGNORED
    at = torch.where(kept, T, 0)[:, None]
    z = X @ W.T
    e = sums(inner) * (X.abs() @ W.abs().T)
    lse = torch.logsumexp(z, 1)
    el = e.amax(1) + U * (8 + 2 * (16 + 4 + vocab / 1024 + 64) + 3 * (z - lse[:, None]).abs().amax(1) * 0.4 + 4 * lse.abs())
    want = torch.where(kept, lse - z.gather(1, at)[:, 0], 0.0)
    room = torch.where(kept, 1.01 * (el + e.gather(1, at)[:, 0] + 2 * U * want.abs()), 0.0)
    n = kept.sum()
    if reduction == "none":
        assert ((loss.double().reshape(-1) - want).abs() <= room).all()
        A = torch.where(kept, a.double(), 0.0)
    else:
        by = n if reduction == "mean" else 1
        assert (loss.double() - want.sum() / by).abs() <= room.sum() / by + U * (want.sum() / by).abs()
        A = torch.where(kept, upstream / by, 0.0).double()
    p = torch.exp(z - lse[:, None])
    G = A[:, None] * p
    eg = G.abs() * (e + el[:, None] + U * (8 + 3 * (z - lse[:, None]).abs()))
    G = G.scatter_add(1, at, -A[:, None])
    eg = 1.01 * (eg + (h + 3 * U) * G.abs() + 2 * U * A.abs()[:, None] * (torch.arange(vocab, device="cuda") == at))
    # times a power of two an fp16 G has its largest weight at 2^13 and steps of 2^-24 at the least
    eg = eg + (2.0 ** -38 * A.abs().max() if x.dtype == F16 else 1e-37)
    pieces = 64  # of the vocabulary at most, each an addition to dx
    want = G @ W
    room = eg @ W.abs() + (sums(vocab) + pieces * 2 * U) * (G.abs() @ W.abs()) + (h + 2 * U) * want.abs() + least
    assert ((dx.double().reshape(rows, inner) - want).abs() <= 1.01 * room).all()
    want = G.T @ X
    room = eg.T @ X.abs() + sums(rows) * (G.abs().T @ X.abs()) + (h + 2 * U) * want.abs() + least
    assert ((dw.double() - want).abs() <= 1.01 * room).all()
    assert (dx.reshape(rows, inner)[~kept] == 0).all()


SHAPES = [(1, 64, 257), (2, 8, 1), (5, 1, 3), (16, 768, 1000), (17, 100, 333), (127, 72, 4099), (128, 64, 256), (129, 1031, 511), (300, 2048, 700), (700, 64, 5003), (257, 1025, 2049)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("rows,inner,vocab", SHAPES)
def test_rows_with_weights(rows, inner, vocab, kind):
    check(*make(rows, inner, vocab, kind, rows + vocab))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 7, 8, 9, 16, 17])
def test_few_rows_over_large_vocabularies(rows, kind):
    for inner, vocab in ((72, 50257), (8, 20001), (1000, 19003), (33, 30000)):
        check(*make(rows, inner, vocab, kind, rows + inner))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("reduction,upstream", [("sum", 1.0), ("mean", 1.0), ("mean", 4096.0), ("sum", 2.0 ** -20), ("mean", 0.0)])
def test_reductions(reduction, upstream, kind):
    check(*make(70, 96, 1003, kind, 5), reduction, upstream)


@pytest.mark.gpu
def test_pieces_of_the_vocabulary():
    """More columns than 384 MiB of G take: 40000 rows, pieces and a rest."""
    x, w, t, a = make(40000, 16, 13001, BF16, 6)
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    loss = ops.linear_cross_entropy(*leaves, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, leaves, a)
    assert _lib.cuda().hc_linear_cross_entropy_backward_bytes(40000, 16, 13001) <= (384 << 20) + 40000 * (4 * 64 + 4) + 1024
    h = torch.finfo(BF16).eps / 2
    W = w.double()
    total = torch.zeros(13001, 16, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(total)
    for i in range(0, 40000, 4000):
        X, T = x[i:i + 4000].double(), t[i:i + 4000]
        kept = T != IGNORED
        at = torch.where(kept, T, 0)[:, None]
        z = X @ W.T
        lse = torch.logsumexp(z, 1, keepdim=True)
        A = torch.where(kept, a[i:i + 4000], 0.0).double()[:, None]
        e = 2 * sums(16) * (X.abs() @ W.abs().T).amax() + 300 * U
        assert (loss[i:i + 4000].double() - torch.where(kept, lse[:, 0] - z.gather(1, at)[:, 0], 0.0)).abs().max() <= e + 8 * U * 20
        G = (A * torch.exp(z - lse)).scatter_add(1, at, -A)
        eg = 1.05 * (h + e) * G.abs() + 2 * U * A.abs() * (torch.arange(13001, device="cuda") == at)
        room = eg @ W.abs() + (sums(13001) + 128 * U) * (G.abs() @ W.abs()) + (h + 2 * U) * (G @ W).abs()
        assert ((dx[i:i + 4000].double() - G @ W).abs() <= 1.01 * room + 1e-37).all()
        total += G.T @ X
        size += eg.T @ X.abs() + sums(40000) * (G.abs().T @ X.abs())
    assert ((dw.double() - total).abs() <= 1.01 * (size + (h + 2 * U) * total.abs())).all()


@pytest.mark.gpu
def test_shapes_and_strides():
    """Rows that begin anywhere, lie apart, or come in more dimensions; weights that are a part of others."""
    x, w, t, a = make(24, 80, 301, BF16, 7)
    wide = torch.zeros(24, 163, dtype=BF16, device="cuda")
    wide[:, 3:83] = x
    broad = torch.zeros(301, 99, dtype=BF16, device="cuda")
    broad[:, 1:81] = w
    check(wide[:, 3:83], w, t, a)
    check(x, broad[:, 1:81], t, a)
    check(x.t().contiguous().t(), w.t().contiguous().t(), t, a)
    check(x.view(2, 3, 4, 80), w, t.view(2, 3, 4), a)
    check(x[:1].expand(24, 80), w, t, a)
    many = torch.stack([t, t], 1)[:, 0]
    check(x, w, many, a)


@pytest.mark.gpu
def test_rows_and_targets_that_have_nothing():
    x, w, t, a = make(9, 64, 130, F16, 8)
    none = torch.full_like(t, IGNORED)
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    assert ops.linear_cross_entropy(x, w, none).isnan() and ops.linear_cross_entropy(x, w, none, reduction="sum") == 0
    for reduction in ("sum", "mean"):
        for g in torch.autograd.grad(ops.linear_cross_entropy(*leaves, none, reduction=reduction), leaves):
            assert (g == 0).all()
    empty = x[:0].detach().requires_grad_()
    for reduction, shape in (("none", (0,)), ("sum", ()), ("mean", ())):
        loss = ops.linear_cross_entropy(empty, leaves[1], t[:0], reduction=reduction)
        assert loss.shape == shape and (reduction != "sum" or loss == 0) and (reduction != "mean" or loss.isnan())
        dx, dw = torch.autograd.grad(loss.sum(), (empty, leaves[1]))
        assert dx.shape == (0, 64) and (dw == 0).all()
    other = t.clone()
    other[3] = 7
    assert torch.equal(ops.linear_cross_entropy(x, w, other, ignore_index=7, reduction="none") == 0, other == 7)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
def test_what_is_not_finite(kind):
    """An ignored row has a loss and a gradient of 0, whatever it holds (the product G^T x has it times 0); a NaN elsewhere shows in its row and in the weights; a target outside of the vocabulary too."""
    x, w, t, a = make(20, 64, 300, kind, 9)
    assert t[3] == IGNORED
    want = [ops.linear_cross_entropy(x, w, t, reduction="none")]
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    want += torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, reduction="none"), leaves, a)
    for bad in (math.nan, math.inf):
        y = x.clone()
        y[3] = bad
        leaves = [v.detach().requires_grad_() for v in (y, w)]
        loss = ops.linear_cross_entropy(*leaves, t, reduction="none")
        got = torch.autograd.grad(loss, leaves, a)
        assert torch.equal(loss, want[0]) and torch.equal(got[0], want[1])
        assert got[1].isnan().all()  # dweight = G^T x: G's zeros times what is not finite
        y = x.clone()
        y[5, 7] = bad
        leaves = [v.detach().requires_grad_() for v in (y, w)]
        loss = ops.linear_cross_entropy(*leaves, t, reduction="none")
        dx, dw = torch.autograd.grad(loss, leaves, a)
        rest = torch.arange(20) != 5
        assert loss[5].isnan() and torch.equal(loss[rest], want[0][rest])
        assert dx[5].isnan().all() and torch.equal(dx[rest], want[1][rest]) and dw[:, 7].isnan().all()
    for outside in (300, -1, 2 ** 40):
        u = t.clone()
        u[5] = outside
        loss = ops.linear_cross_entropy(*leaves, u, reduction="none")
        assert loss[5].isnan()
        y = [v.detach().requires_grad_() for v in (x, w)]
        loss = ops.linear_cross_entropy(*y, u, reduction="none")
        dx, dw = torch.autograd.grad(loss, y, a)
        rest = torch.arange(20) != 5
        assert loss[5].isnan() and torch.equal(loss[rest], want[0][rest]) and dx[5].isnan().all() and torch.equal(dx[rest], want[1][rest]) and dw.isnan().all()


@pytest.mark.gpu
def test_large_logits():
    """Logits in the hundreds: exponentials are taken relative to the row's largest."""
    x, w, t, a = make(40, 128, 513, BF16, 10, scale=60.0)
    check(x, w, t, a)


@pytest.mark.gpu
def test_against_differences():
    """The gradient along a direction against the loss at two places (their difference has an error of the losses over the distance)."""
    x, w, t, _ = make(33, 64, 200, BF16, 11)
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, reduction="sum"), leaves)

    def exact(x, w):
        z = x @ w.T
        kept = t != IGNORED
        return torch.where(kept, torch.logsumexp(z, 1) - z.gather(1, torch.where(kept, t, 0)[:, None])[:, 0], 0.0).sum()

    g = torch.Generator().manual_seed(12)
    for i, (leaf, d) in enumerate(((x, dx), (w, dw))):
        v = torch.randn(leaf.shape, generator=g).double().cuda()
        step = 1e-5
        moved = [[x.double(), w.double()] for _ in range(2)]
        moved[0][i] = moved[0][i] + step * v
        moved[1][i] = moved[1][i] - step * v
        slope = (exact(*moved[0]) - exact(*moved[1])) / (2 * step)
        # each value of the gradient is off by at most three half steps of itself (of G, of the result, and the sums), the direction's values are independent: five sigma
        room = 5 * 3 * 2.0 ** -8 * d.double().norm() + 1e-6
        assert (slope - (d.double() * v).sum()).abs() <= room


@pytest.mark.gpu
def test_captured_and_on_two_streams():
    """Two graphs, each with scratch memory of its own, replayed at once on other values."""
    sets = [make(200, 96, 3001, BF16, 20 + i) for i in range(2)]
    graphs, outs, held = [], [], []
    for x, w, t, a in sets:
        leaves = [v.clone().requires_grad_() for v in (x, w)]
        held.append((leaves, t, a))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, reduction="none"), leaves, a)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = ops.linear_cross_entropy(*leaves, t, reduction="none")
            grads = torch.autograd.grad(loss, leaves, a)
        graphs.append(graph)
        outs.append((loss, *grads))
    with torch.no_grad():
        for (leaves, t, a), other in zip(held, sets[::-1]):
            for u, v in zip((*leaves, t, a), other):
                u.copy_(v)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for (leaves, t, a), got in zip(held, outs):
        fresh = [v.detach().clone().requires_grad_() for v in leaves]
        loss = ops.linear_cross_entropy(*fresh, t, reduction="none")
        want = (loss, *torch.autograd.grad(loss, fresh, a))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert ops.train_status() == 0


def _good(device):
    return [torch.zeros(4, 16, dtype=BF16, device=device), torch.zeros(9, 16, dtype=BF16, device=device), torch.zeros(4, dtype=torch.int64, device=device)]


@pytest.mark.gpu
def test_refusals():
    x, w, t = _good("cuda")
    for args, kw in (((x.float(), w, t), {}), ((x, w.half(), t), {}), ((x, w[:, :8], t), {}), ((x, w, t.int()), {}), ((x, w, t[:3]), {}), ((x, w, t), dict(reduction="max")),
                     ((x, w[:0], t), {}), ((x, w.cpu(), t), {}), ((x, w, t.cpu()), {}), ((x[0, 0], w, t), {})):
        with pytest.raises(ValueError):
            ops.linear_cross_entropy(*args, **kw)
    leaf = x.clone().requires_grad_()
    (d,) = torch.autograd.grad(ops.linear_cross_entropy(leaf, w, t), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradients of their own"):
        d.sum().backward()
    neg = torch._neg_view(w.clone())
    assert torch.equal(ops.linear_cross_entropy(x + 1, neg, t), ops.linear_cross_entropy(x + 1, -w, t))


def test_refusals_without_a_gpu():
    import torch.autograd.forward_ad as forward_ad

    x, w, t = _good("cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_cross_entropy(x, w, t)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            ops.linear_cross_entropy(forward_ad.make_dual(x, torch.ones_like(x)), w, t)
    with pytest.raises(NotImplementedError):
        torch.vmap(lambda v: ops.linear_cross_entropy(v, w, t))(torch.stack([x, x]))


def test_c_entry_points_refuse():
    """Nothing below is launched."""
    lib = _lib.cuda()
    p, odd, half, some = (C.c_void_p(v) for v in (4096, 4097, 4098, 4112))
    big = 1 << 40
    forward = dict(x=p, xs=16, w=p, ws=16, type=1, t=p, ig=-100, red=0, loss=p, stats=p, m=4, k=16, n=24, scratch=p, bytes=big)
    backward = dict(x=p, xs=16, w=p, ws=16, type=1, t=p, ig=-100, red=0, stats=p, dl=p, dx=p, dxs=16, dw=p, dws=16, m=4, k=16, n=24, scratch=p, bytes=big)
    both = [dict(x=None), dict(x=half), dict(w=half), dict(xs=15), dict(xs=20), dict(ws=20), dict(ws=8), dict(type=0), dict(type=3), dict(red=3), dict(red=-1), dict(t=None), dict(t=some.value + 4), dict(stats=None),
            dict(stats=half), dict(m=1 << 26), dict(k=1 << 26), dict(n=1 << 26), dict(k=0), dict(n=0), dict(scratch=None), dict(scratch=some)]
    for bad in both + [dict(loss=None), dict(loss=half), dict(bytes=10)]:
        assert lib.hc_linear_cross_entropy(*{**forward, "m": 40, **bad}.values(), None) == 4, bad
    for bad in (dict(x=odd), dict(w=odd), dict(xs=15), dict(bytes=10)):  # few rows may begin anywhere
        assert lib.hc_linear_cross_entropy(*{**forward, **bad}.values(), None) == 4, bad
    for bad in both + [dict(dl=None), dict(dl=half), dict(dx=odd), dict(dw=odd), dict(dxs=8), dict(dws=15), dict(bytes=10)]:
        assert lib.hc_linear_cross_entropy_backward(*{**backward, **bad}.values(), None) == 4, bad
    assert lib.hc_linear_cross_entropy_backward(*{**backward, "dx": None, "dw": None}.values(), None) == 0
    assert lib.hc_linear_cross_entropy_bytes(0, 16, 24) == 0 and lib.hc_linear_cross_entropy_bytes(4, 1 << 26, 24) == 0


def test_scratch_memory_is_bounded():
    lib = _lib.cuda()
    for rows, inner, vocab in ((8192, 768, 50257), (1, 4096, 131072), (100000, 64, 131072), (300000, 8, 5000), (1 << 20, 8, 1025)):
        g = max(384 << 20, rows * 1024 * 2)
        assert lib.hc_linear_cross_entropy_backward_bytes(rows, inner, vocab) <= g + 4 * rows * (inner + 8) * 4 + rows * 4 + 2048
        assert lib.hc_linear_cross_entropy_bytes(rows, inner, vocab) <= rows * ((vocab + 63) // 64 * 32 + 8) + 2048


@pytest.mark.gpu
def test_model_without_logits():
    """The model's loss and gradients from hidden rows against the same model with its logits, in 64 bits: 40 roundings of at most 2^-8, as for the model with logits."""
    import copy

    import torch.nn.functional as F

    cfg = GPT2Config.tiny()
    torch.manual_seed(0)
    plain = GPT2(cfg).cuda()
    cfg = copy.copy(cfg)
    cfg.fused, cfg.logits = True, False
    fused = GPT2(cfg).cuda()
    fused.load_state_dict(plain.state_dict())
    plain = plain.double()
    tok = torch.randint(0, 257, (3, 33), generator=torch.Generator().manual_seed(1)).cuda()
    idx, targets = tok[:, :-1], tok[:, 1:].clone()
    targets[0, :5] = -100
    loss = fused(idx, targets)
    loss.backward()
    want = plain(idx)
    exact = F.cross_entropy(want.reshape(-1, 257), targets.reshape(-1))
    exact.backward()
    room = 40 * 2.0 ** -8
    assert abs(loss.item() - exact.item()) <= room * exact.item()
    for (name, p), q in zip(fused.named_parameters(), plain.parameters()):
        scale = q.grad.norm() if not name.endswith("qkv.bias") else fused.blocks[0].qkv.weight.grad.double().norm()
        assert (p.grad.double() - q.grad).norm() <= room * scale, name
    assert fused(idx).shape == (3, 32, 257)
    assert ops.train_status() == 0
