"""Attention and its gradients against the formulas in 64 bits.

Tolerances count roundings.  u and h are half a step of fp32 and of the operands' type.  A score is a sum over the head's values, whose products are exact in fp32, through at most d / 16 + 20
additions, each off by at most a whole step; an exponential is off by its argument's error and 4 u.  Probabilities are rounded to the operands' type (h) before they enter the product with the
values; in fp16 those below 2^-24 of a row's reference are lost, 2^-31 of the row's sum each.  The backward pass forms probabilities again in the same way; delta is the product of dO with the rounded O;
dS is rounded (h), in fp16 times a power of two with which 2 max|dO| max|V| is at least 2^12, so that no more than 2^-37 of that is lost."""
import ctypes as C
import math

import pytest
import torch

from tirocinio_triennale_b200 import _lib, ops
from tirocinio_triennale_b200._lib_train import Heads
from tirocinio_triennale_b200.models import GPT2, GPT2Config

U = torch.finfo(torch.float32).eps / 2
BF16, F16 = torch.bfloat16, torch.float16


def sums(k):
    return (k / 16 + 20) * 2 * U


def make(batch, heads, kv_heads, queries, keys, d, kind, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)

    def some(n, h):
        return (scale * torch.randn(batch, n, h, d, generator=g)).to(kind).cuda().transpose(1, 2)

    return some(queries, heads), some(keys, kv_heads), some(keys, kv_heads), (some(queries, heads) / scale).to(kind)


def seen_by(queries, keys, window, sinks):
    p = torch.arange(queries, device="cuda")[:, None] + keys - queries
    j = torch.arange(keys, device="cuda")[None]
    seen = j <= p
    return seen if window is None else seen & ((p - j < window) | (j < sinks))


def check(q, k, v, dout, window=None, sinks=0, scale=None, grads=True):
    kind, (b, heads, m, d), kv, n = q.dtype, q.shape, k.shape[1], k.shape[2]
    h, least = torch.finfo(kind).eps / 2, 2.0 ** -25 if kind == F16 else 1e-37
    f16 = kind == F16
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    kw = dict(window=window, sinks=sinks, scale=scale)
    o = ops.attention(*leaves, **kw)
    assert o.shape == q.shape and o.dtype == kind and o.transpose(1, 2).is_contiguous()
    again = ops.attention(q, k, v, **kw)
    assert torch.equal(o, again) or (o != o).any()
    c = scale or 1 / math.sqrt(d)
    group = heads // kv
    Q, D = q.double().reshape(b, kv, group, m, d), dout.double().reshape(b, kv, group, m, d)
    K, V = k.double()[:, :, None], v.double()[:, :, None]
    seen = seen_by(m, n, window, sinks)
    s = c * (Q @ K.mT)
    es = c * sums(d) * (Q.abs() @ K.abs().mT) + 3 * U * s.abs()
    s = s.masked_fill(~seen, -math.inf)
    some = seen.any(1)
    top = torch.where(some, s.amax(-1), 0.0)
    p = torch.exp(s - top[..., None])
    p = p / torch.where(some, p.sum(-1), 1.0)[..., None]
    E = torch.where(seen, es, 0.0).amax(-1) + U * (40 + 4 * top.abs() + 4 * torch.where(seen & (p > 1e-8), (s - top[..., None]).abs(), 0.0).amax(-1) + n / 128)
    O = p @ V
    room_o = (2 * E + h + sums(n))[..., None] * (p @ V.abs()) + (h + 4 * U) * O.abs() + least
    if f16:
        room_o = room_o + 2.0 ** -30 * (seen.double() @ V.abs())
    room_o = torch.where(some[:, None], 1.02 * room_o, 0.0)
    got = o.double().reshape(b, kv, group, m, d)
    assert ((got - O).abs() <= room_o).all(), float(((got - O).abs() - room_o).max())
    if not grads:
        return
    dq, dk, dv = torch.autograd.grad(o, leaves, dout)
    for t, leaf in zip((dq, dk, dv), leaves):
        assert t.shape == leaf.shape and t.dtype == kind and t.transpose(1, 2).is_contiguous()
    dp = D @ V.mT
    delta = (D * O).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    off = sums(d) * (D.abs() @ V.abs().mT) + (D.abs() * room_o).sum(-1, keepdim=True) + (20 * U) * (D.abs() * O.abs()).sum(-1, keepdim=True)
    eds = p * (2 * E[..., None] * (dp - delta).abs() + off) + (h + 4 * U) * ds.abs()
    ep = (2 * E[..., None] + h) * p
    if f16:
        size = 2 * D.norm(dim=-1).amax() * V.norm(dim=-1).amax()
        eds = eds + 2.0 ** -36 * size * seen
        ep = ep + 2.0 ** -38 * seen
    room = c * (eds @ K.abs() + sums(n) * (ds.abs() @ K.abs())) + (h + 4 * U) * (c * (ds @ K)).abs() + least
    got = dq.double().reshape(b, kv, group, m, d)
    assert ((got - c * (ds @ K)).abs() <= 1.02 * room).all(), float(((got - c * (ds @ K)).abs() - room).max())
    want = c * (ds.mT @ Q).sum(2)
    room = c * (eds.mT @ Q.abs() + sums(m * group) * (ds.abs().mT @ Q.abs())).sum(2) + (h + 4 * U) * want.abs() + least
    assert ((dk.double() - want).abs() <= 1.02 * room).all(), float(((dk.double() - want).abs() - room).max())
    want = (p.mT @ D).sum(2)
    room = (ep.mT @ D.abs() + sums(m * group) * (p.mT @ D.abs())).sum(2) + (h + 4 * U) * want.abs() + least
    assert ((dv.double() - want).abs() <= 1.02 * room).all(), float(((dv.double() - want).abs() - room).max())
    for i, t in enumerate((dq, dk, dv)):  # one alone
        leaves = [x.detach().requires_grad_(j == i) for j, x in enumerate((q, k, v))]
        (one,) = torch.autograd.grad(ops.attention(*leaves, **kw), leaves[i], dout)
        assert torch.equal(one, t)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("d", [8, 32, 64, 80, 128])
@pytest.mark.parametrize("length", [1, 2, 127, 128, 129, 257, 640])
def test_whole_sequences(length, d, kind):
    check(*make(2, 3, 3, length, length, d, kind, length + d))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 3), (64, 0), (127, 4), (128, 0), (129, 130), (300, 1), (300, 600), (5000, 7)])
def test_windows_and_sinks(window, sinks, kind):
    check(*make(1, 4, 2, 701, 701, 64, kind, window + sinks), window=window, sinks=sinks)
    check(*make(1, 2, 1, 333, 900, 128, kind, window + sinks), window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (2, 1), (6, 2), (5, 5), (40, 8), (12, 1)])
@pytest.mark.parametrize("queries,keys", [(1, 1), (1, 300), (3, 3000), (16, 77), (130, 515), (20, 7), (300, 130), (3, 1)])
def test_chunks_and_shared_heads(queries, keys, heads, kv_heads, kind):
    """New tokens behind others, queries in front of the first key (which see nothing), query heads that share keys."""
    check(*make(2, heads, kv_heads, queries, keys, 64, kind, queries + keys))
    check(*make(1, heads, kv_heads, queries, keys, 96, kind, queries + keys), window=40, sinks=2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
def test_single_tokens_behind_long_texts(kind):
    """Keys shared out to several CTAs."""
    for batch, heads, kv, keys, d, window, sinks in ((1, 12, 12, 1024, 64, None, 0), (2, 8, 2, 9001, 128, None, 0), (1, 4, 1, 20000, 128, 4096, 4), (3, 6, 3, 5000, 72, 130, 1), (1, 1, 1, 30011, 64, None, 0)):
        check(*make(batch, heads, kv, 1, keys, d, kind, keys), window=window, sinks=sinks, grads=False)
        check(*make(batch, heads, kv, 7, keys, d, kind, keys), window=window, sinks=sinks, grads=keys < 10000)


@pytest.mark.gpu
def test_long_rows_of_many_tiles():
    check(*make(1, 2, 1, 3000, 3000, 64, BF16, 1))
    check(*make(1, 2, 2, 2500, 2500, 128, F16, 2), window=1000, sinks=130)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
def test_large_and_small_scores(kind):
    """Scores in the hundreds, of one sign and of both; rows whose largest score grows from tile to tile; uniform rows."""
    q, k, v, dout = make(1, 2, 2, 500, 500, 64, kind, 3, scale=5.0)
    check(q, k, v, dout)
    check(q, k, v, dout, scale=1e-3)
    grow = (torch.arange(500, device="cuda").view(1, 1, 500, 1) / 50).to(kind)
    check(torch.ones_like(q), (grow * torch.ones_like(k)).to(kind), v, dout)
    check(torch.ones_like(q), (-grow * torch.ones_like(k)).to(kind), v, dout)
    check(torch.zeros_like(q), k, v, dout)


@pytest.mark.gpu
def test_small_gradients_in_fp16():
    """Upstream gradients whose dS would be nothing in fp16 without its power of two."""
    q, k, v, dout = make(1, 2, 1, 400, 400, 64, F16, 4)
    check(q, k, v, (dout * 1e-4).to(F16))
    check(q, k, (v * 100).to(F16), (dout * 60).to(F16))
    check(q, k, v, torch.zeros_like(dout))


@pytest.mark.gpu
def test_views_and_strides():
    """Parts of a projection's result are read where they lie; what the kernels cannot read is copied."""
    g = torch.Generator().manual_seed(5)
    joint = torch.randn(2, 200, 3 * 4 * 64, generator=g).to(BF16).cuda()
    q, k, v = (t.view(2, 200, 4, 64).transpose(1, 2) for t in joint.split(256, 2))
    dout = torch.randn(2, 4, 200, 64, generator=g).to(BF16).cuda()
    check(q, k, v, dout)
    check(q.contiguous(), k.contiguous(), v.contiguous(), dout)
    odd = torch.randn(2, 200, 3 * 4 * 64 + 3, generator=g).to(BF16).cuda()
    a, b, c = (odd[..., i * 256 + 1:i * 256 + 257].reshape(2, 200, 4, 64).transpose(1, 2) if i == 0 else odd[..., i * 256 + 1:i * 256 + 257].unflatten(2, (4, 64)).transpose(1, 2) for i in range(3))
    check(a, b, c, dout)
    check(q, k[:, :1].expand(2, 4, 200, 64), v[:, :1].expand(2, 4, 200, 64), dout[:1].expand(2, 4, 200, 64))
    last = torch.randn(2, 4, 64, 200, generator=g).to(BF16).cuda().transpose(2, 3)
    check(last, k, v, dout.transpose(2, 3).contiguous().transpose(2, 3))
    check(q[:, :, ::2], k[:, :, ::2], v[:, :, ::2], dout[:, :, ::2])
    check(q[:, ::2], k[:, ::2], v[:, ::2], dout[:, ::2])


@pytest.mark.gpu
def test_nothing_to_do():
    q, k, v, dout = make(2, 2, 2, 5, 7, 64, BF16, 6)
    none = k[:, :, :0]
    leaves = [t.detach().requires_grad_() for t in (q, none, none)]
    o = ops.attention(*leaves)
    assert (o == 0).all()
    dq, dk, dv = torch.autograd.grad(o, leaves, dout)
    assert (dq == 0).all() and dk.shape == dv.shape == none.shape
    for a, b in ((q[:, :, :0], k), (q[:0], k[:0])):
        leaves = [t.detach().requires_grad_() for t in (a, b, b)]
        o = ops.attention(*leaves)
        assert o.shape == a.shape
        dq, dk, dv = torch.autograd.grad(o.sum(), leaves)
        assert dq.shape == a.shape and (dk == 0).all() and (dv == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
def test_what_is_not_finite(kind):
    """It shows where it is seen, and in no other head or sequence."""
    q, k, v, dout = make(2, 4, 2, 300, 300, 64, kind, 7)
    want = ops.attention(q, k, v, window=50, sinks=2)
    for bad in (math.nan, math.inf):
        for which in range(3):
            inputs = [t.clone() for t in (q, k, v)]
            inputs[which][1, 1, 200, 3] = bad
            o = ops.attention(*inputs, window=50, sinks=2)
            heads = [1] if which == 0 else [2, 3]
            for b in range(2):
                for h in range(4):
                    if b == 0 or h not in heads:
                        assert torch.equal(o[b, h], want[b, h])
            if which == 0:
                assert o[1, 1, 200].isnan().all() and torch.equal(o[1, 1, :200], want[1, 1, :200]) and torch.equal(o[1, 1, 201:], want[1, 1, 201:])
            elif which == 2:
                assert not o[1, 2, 200:250, 3].isfinite().any()
            elif bad != bad:
                assert o[1, 2, 200:250].isnan().all()
    masked = k.clone()
    masked[:, :, 299] = math.nan  # a key in the future: its score is masked
    assert torch.equal(ops.attention(q, masked, v)[:, :, :299], ops.attention(q, k, v)[:, :, :299])


@pytest.mark.gpu
def test_against_differences():
    """The gradient along a direction against the formula's difference at two places: each value is off by some four half steps of its own, independently; five sigma."""
    q, k, v, dout = make(1, 4, 2, 150, 200, 64, BF16, 8)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.attention(*leaves, window=60, sinks=3), leaves, dout)
    seen = seen_by(150, 200, 60, 3)

    def exact(q, k, v):
        s = (q.view(1, 2, 2, 150, 64) @ k[:, :, None].mT / 8).masked_fill(~seen, -math.inf)
        return ((torch.softmax(s, -1) @ v[:, :, None]).view(1, 4, 150, 64) * dout.double()).sum()

    g = torch.Generator().manual_seed(9)
    for i, d in enumerate(grads):
        way = torch.randn(d.shape, generator=g).double().cuda()
        moved = [[t.double().contiguous() for t in (q, k, v)] for _ in range(2)]
        moved[0][i] = moved[0][i] + 1e-5 * way
        moved[1][i] = moved[1][i] - 1e-5 * way
        slope = (exact(*moved[0]) - exact(*moved[1])) / 2e-5
        assert (slope - (d.double() * way).sum()).abs() <= 5 * 4 * 2.0 ** -8 * d.double().norm()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
def test_captured_and_on_two_streams(kind):
    """Two graphs replayed at once on other values, each with scratch memory of its own; single tokens and sequences."""
    sets = [(make(2, 4, 2, 1, 5000, 64, kind, 10 + i), make(1, 4, 4, 300, 300, 64, kind, 20 + i)) for i in range(2)]
    graphs, outs, held = [], [], []

    def call(token, whole):
        leaves = whole[:3]
        o = ops.attention(*leaves, window=100, sinks=1)
        return (ops.attention(*token[:3]), o, *torch.autograd.grad(o, leaves, whole[3]))

    for token, whole in sets:
        token = [t.clone() for t in token]
        whole = [t.clone().requires_grad_(i < 3) for i, t in enumerate(whole)]
        held.append((token, whole))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(token, whole)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(token, whole))
        graphs.append(graph)
    with torch.no_grad():
        for (token, whole), (other, theirs) in zip(held, sets[::-1]):
            for a, b in zip((*token, *whole), (*other, *theirs)):
                a.copy_(b)
    torch.cuda.synchronize()
    for g, s in zip(graphs, [torch.cuda.Stream() for _ in range(2)]):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for (token, whole), got in zip(held, outs):
        want = call(token, [t.detach().clone().requires_grad_(i < 3) for i, t in enumerate(whole)])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert ops.train_status() == 0


def _good(device):
    return [torch.zeros(2, 4, 3, 16, dtype=BF16, device=device), torch.zeros(2, 2, 5, 16, dtype=BF16, device=device), torch.zeros(2, 2, 5, 16, dtype=BF16, device=device)]


@pytest.mark.gpu
def test_refusals():
    q, k, v = _good("cuda")
    for args, kw in (((q.float(), k, v), {}), ((q, k.half(), v), {}), ((q.float(), k.float(), v.float()), {}), ((q[0], k, v), {}), ((q, k, v[:, :1]), {}), ((q[:1], k, v), {}), ((q[..., :8], k, v), {}),
                     ((q[:, :3], k, v), {}), ((q, k[:, :0], v[:, :0]), {}), ((q[..., :12], k[..., :12], v[..., :12]), {}), ((q, k, v), dict(window=0)), ((q, k, v), dict(window=-3)), ((q, k, v), dict(sinks=-1)),
                     ((q, k, v), dict(scale=0.0)), ((q, k, v), dict(scale=-1.0)), ((q, k, v), dict(scale=math.inf)), ((q, k, v), dict(scale=math.nan)), ((q, k.cpu(), v), {}),
                     ((torch.zeros(1, 1, 2, 136, dtype=BF16, device="cuda"),) * 3, {})):
        with pytest.raises(ValueError):
            ops.attention(*args, **kw)
    leaf = q.clone().requires_grad_()
    (d,) = torch.autograd.grad(ops.attention(leaf, k, v).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="no gradients of their own"):
        d.sum().backward()
    q, k, v, dout = make(1, 2, 2, 20, 20, 64, BF16, 30)
    assert torch.equal(ops.attention(q, torch._neg_view(k), v), ops.attention(q, -k, v))


def test_refusals_without_a_gpu():
    import torch.autograd.forward_ad as forward_ad

    q, k, v = _good("cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention(q, k, v)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            ops.attention(forward_ad.make_dual(q, torch.ones_like(q)), k, v)
    with pytest.raises(NotImplementedError):
        torch.vmap(lambda t: ops.attention(t, k, v))(torch.stack([q, q]))


def test_c_entry_points_refuse():
    """Nothing below is launched."""
    lib = _lib.cuda()
    p, half, some, big = C.c_void_p(4096), C.c_void_p(4098), C.c_void_p(4104), 1 << 40

    def at(data=4096, batch=4096, head=1024, position=16):
        return Heads(data, batch, head, position)

    forward = dict(q=at(), k=at(), v=at(), type=1, out=p, stats=p, b=2, h=4, kv=2, m=3, n=5, d=16, w=0, s=0, scale=0.25)
    backward = dict(do=at(), out=p, q=at(), k=at(), v=at(), type=1, stats=p, dq=p, dk=p, dv=p, b=2, h=4, kv=2, m=3, n=5, d=16, w=0, s=0, scale=0.25, scratch=p, bytes=big)
    both = [dict(q=at(data=4098)), dict(k=at(data=None)), dict(v=at(position=12)), dict(q=at(position=8)), dict(k=at(head=1028)), dict(v=at(batch=0)), dict(type=0), dict(type=3), dict(out=None), dict(out=some),
            dict(stats=some), dict(h=3), dict(kv=0), dict(m=1 << 24), dict(n=1 << 24), dict(d=12), dict(d=136), dict(d=0), dict(b=1 << 24), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)]
    for bad in both:
        assert lib.hc_attention(*{**forward, **bad}.values(), None) == 4, bad
    for bad in both + [dict(do=at(data=4098)), dict(stats=None), dict(dk=None), dict(dv=None), dict(dq=half), dict(scratch=None), dict(scratch=some), dict(bytes=16)]:
        assert lib.hc_attention_backward(*{**backward, **bad}.values(), None) == 4, bad
    assert lib.hc_attention_backward(*{**backward, "dq": None, "dk": None, "dv": None}.values(), None) == 0
    assert lib.hc_attention(*{**forward, "b": 0}.values(), None) == 0 and lib.hc_attention(*{**forward, "m": 0}.values(), None) == 0
    assert lib.hc_attention_backward_bytes(2, 3, 2, 3, 5, 16) == 0 and lib.hc_attention_stats(2, 4, 129) == 2 * 4 * 256


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [dict(window=8, sinks=2), dict(d_model=96, n_head=3, vocab_size=1001, n_layer=1, logits=False), dict(d_model=128, n_head=2, window=5, attention="own")])
def test_model_with_this_attention(shape):
    """The model through this library's attention, with a window, against its formulas in 64 bits: 40 roundings of at most 2^-8, as without."""
    import copy

    import torch.nn.functional as F

    cfg = GPT2Config.tiny()
    for name, value in shape.items():
        setattr(cfg, name, value)
    cfg.attention = "own"
    torch.manual_seed(0)
    plain_cfg = copy.copy(cfg)
    plain_cfg.attention = "torch"
    plain = GPT2(plain_cfg).cuda()
    cfg.fused = True
    fused = GPT2(cfg).cuda()
    fused.load_state_dict(plain.state_dict())
    plain = plain.double()
    tok = torch.randint(0, cfg.vocab_size, (3, 33), generator=torch.Generator().manual_seed(1)).cuda()
    idx, targets = tok[:, :-1], tok[:, 1:].clone()
    targets[0, :5] = -100
    loss = fused(idx, targets)
    loss.backward()
    want = plain(idx)
    exact = F.cross_entropy(want.reshape(-1, want.shape[-1]), targets.reshape(-1))
    exact.backward()
    room = 40 * 2.0 ** -8
    assert abs(loss.item() - exact.item()) <= room * exact.item()
    for (name, p), q in zip(fused.named_parameters(), plain.parameters()):
        scale = q.grad.norm() if not name.endswith("qkv.bias") else fused.blocks[0].qkv.weight.grad.double().norm()
        assert (p.grad.double() - q.grad).norm() <= room * scale, name
    assert ops.train_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,queries,d", [(16, 16, 1, 128), (16, 1, 1, 128), (16, 2, 2, 96), (12, 12, 1, 64), (24, 2, 1, 64)])
def test_many_calls_give_the_same(heads, kv_heads, queries, d):
    """Long runs of steps by all of the GPU, again and again: the same bits, and no wait that runs out."""
    g = torch.Generator("cuda").manual_seed(7)
    q = torch.randn(32, heads, queries, d, dtype=BF16, device="cuda", generator=g)
    k, v = (torch.randn(32, kv_heads, 4099, d, dtype=BF16, device="cuda", generator=g) for _ in range(2))
    first = ops.attention(q, k, v)
    assert first.isfinite().all()
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(200):
        differ += (ops.attention(q, k, v) != first).any()
    assert differ.item() == 0
    assert ops.train_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("d", [8, 64, 72, 128])
@pytest.mark.parametrize("heads,kv_heads,queries", [(1, 1, 1), (8, 1, 1), (3, 1, 2), (4, 2, 3), (2, 2, 7), (4, 4, 8), (14, 2, 1)])
def test_up_to_eight_rows(heads, kv_heads, queries, d, kind):
    """Lengths around what a warp, a CTA and a cluster load at once; queries in front of the first key; windows whose gap begins anywhere."""
    for n, (keys, window, sinks) in enumerate([(1, None, 0), (3, 2, 1), (16, None, 0), (17, 5, 2), (127, 1, 0), (129, None, 0), (300, 130, 17), (1025, 1000, 3), (1040, 40, 40), (5003, None, 0), (5003, 300, 20)]):
        q, k, v, dout = make(2, heads, kv_heads, queries, keys, d, kind, n)
        check(q, k, v, dout, window, sinks, grads=n % 3 == 0)


@pytest.mark.gpu
def test_few_rows_of_many_texts():
    """More texts and heads than the second dimension of a grid holds."""
    g = torch.Generator("cuda").manual_seed(3)
    q, k, v = (torch.randn(70000, 2, n, 8, dtype=BF16, device="cuda", generator=g) for n in (1, 3, 3))
    p = torch.softmax(q.double() @ k.double().transpose(2, 3) / math.sqrt(8), 3)
    want = p @ v.double()
    h = torch.finfo(BF16).eps / 2
    # a score's sum of 8 in 32 bits moves a probability by less than 2^-18 of itself; it is rounded for the product, and the result once
    room = (h + 2.0 ** -17) * (p @ v.double().abs()) + h * want.abs() * (1 + 2 * h) + 1e-30
    assert ((ops.attention(q, k, v).double() - want).abs() <= room).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,length,d", [(12, 12, 500, 64), (8, 4, 700, 128), (2, 2, 100, 64)])
def test_many_backward_passes_give_the_same(heads, kv_heads, length, d, kind):
    """Kernels that begin beside the one before them: the same bits again and again, with other values in the memory that they take and other work before and behind them."""
    q, k, v, dout = make(4, heads, kv_heads, length, length, d, kind, 9)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    first = [t.clone() for t in torch.autograd.grad(ops.attention(*leaves), leaves, dout)]
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(100):
        scratch = [torch.full((1 << n,), math.nan, device="cuda") for n in (14, 16, 18, 20)]
        del scratch
        if i % 3 == 2:
            (dq,) = torch.autograd.grad(ops.attention(*leaves), leaves[:1], dout)
            differ += (dq != first[0]).any()
            continue
        for a, b in zip(torch.autograd.grad(ops.attention(*leaves), leaves, dout), first):
            differ += (a != b).any()
    assert differ.item() == 0
    assert ops.train_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [2, 12])
def test_offsets_beyond_32_bits(heads):
    """The end of a cache of 2^24 - 64 positions of two texts, 2^32 values and more, against its last positions alone: the same bits."""
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 20 GB")
    n, m = (1 << 24) - 64, 1024
    k, v = (torch.zeros(2, 1, n, 128, dtype=BF16, device="cuda") for _ in range(2))
    g = torch.Generator("cuda").manual_seed(1)
    q = torch.randn(2, heads, 1, 128, dtype=BF16, device="cuda", generator=g)
    for t in (k, v):
        t[:, :, -m:] = torch.randn(2, 1, m, 128, dtype=BF16, device="cuda", generator=g)
    want = ops.attention(q, k[:, :, -m:].contiguous(), v[:, :, -m:].contiguous(), window=700)
    assert torch.equal(ops.attention(q, k, v, window=700), want)
    assert want.norm() > 0
