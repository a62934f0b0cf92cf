"""The AdamW step against its formulas in 64 bits: moments in 32 bits, moments in 8 bits, the optimiser and the trainer that use it."""
import argparse
import copy
import ctypes as C

import pytest
import torch

from mp_util import run_ranks
from tirocinio_triennale_b200 import _lib, ops
from tirocinio_triennale_b200.models import GPT2, AdamW, GPT2Config, muon_with_adamw

U = 2.0 ** -24  # half a step of fp32
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def _random(seed):
    return torch.Generator().manual_seed(seed)


def _exact(p, g, m, v, step, lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1):
    """The step in 64 bits, and how far fp32 may be from it: every operation is off by U of its result, every constant by U of itself."""
    p, g, m, v = p.double(), g.double(), m.double(), v.double()
    b1, b2 = betas
    terms = (b1 * m).abs() + ((1 - b1) * g).abs()
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    below = (v1 / (1 - b2 ** step)).sqrt() + eps
    size = lr / (1 - b1 ** step)
    p1 = p * (1 - lr * weight_decay) - size * m1 / below
    # m: two constants, two products, a sum; v the same and a square; the parameter besides: a root, two constants, two products, two sums, a quotient
    return p1, m1, v1, 5 * U * terms, 5 * U * v1 + 2.0 ** -148, 4 * U * p.abs() + 16 * U * size * terms / below


def _within(got, want, room):
    off = (got.double() - want).abs()
    assert got.isfinite().all() and (off <= room).all(), float((off - room).max())


def _step_of_code(value, scale, fraction, top):
    """The distance between neighbouring codes around `value`: they stand for 2^e (1 + f) scale / top, e from -15 to -1."""
    e = torch.floor(torch.log2((value / scale * top).clamp(min=2.0 ** -30))).clamp(min=-15)
    return torch.exp2(e - fraction) * scale / top


def _state(n, bits, seed, like=None):
    g = _random(seed)
    if bits == 32:
        return 3e-3 * torch.randn(n, generator=g).cuda(), (1e-2 * torch.rand(n, generator=g)).square().cuda(), None
    return (torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8).cuda(), torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8).cuda(),
            (1e-3 * torch.rand((n + 255) // 256, 2, generator=g) + 1e-6).cuda())


SIZES = [1, 2, 7, 8, 255, 256, 257, 511, 4096, 65537]


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("param,grad", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_moments_in_32_bits(param, grad, shift):
    """Tensors of all sizes that begin `shift` values behind a boundary; what lies between them stays."""
    step = 3
    g = _random(1)
    total = sum(n + shift + 16 for n in SIZES)
    flat = [0.1 * torch.randn(total, generator=g), 0.01 * torch.randn(total, generator=g), 3e-3 * torch.randn(total, generator=g), (1e-2 * torch.rand(total, generator=g)).square()]
    flat = [t.to(k).cuda() for t, k in zip(flat, (param, grad, torch.float32, torch.float32))]
    kept = [t.clone() for t in flat]
    at, places = 0, []
    for n in SIZES:
        places.append(slice(at + shift, at + shift + n))
        at += (n + shift + 15) // 16 * 16
    lists = [[t[s] for s in places] for t in flat]
    ops.adamw_step(*lists, step=step, **HYPER)
    between = torch.ones(total, dtype=torch.bool)
    for i, s in enumerate(places):
        between[s] = False
        p1, m1, v1, rm, rv, rp = _exact(*(t[s] for t in kept), step, **HYPER)
        _within(lists[2][i], m1, rm)
        _within(lists[3][i], v1, rv)
        if param != torch.float32:
            rp = rp + torch.finfo(param).eps / 2 * p1.abs() + torch.finfo(param).smallest_normal * torch.finfo(param).eps
        _within(lists[0][i], p1, rp)
        assert torch.equal(flat[1][s], kept[1][s])
    for t, k in zip(flat, kept):
        assert torch.equal(t[between.cuda()], k[between.cuda()])


@pytest.mark.gpu
def test_values_of_all_codes():
    """Codes are numbers with 4 bits of exponent, the lowest of them without a leading one; scale times the number over the largest one."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    scales = torch.tensor([[3.0, 0.5]], device="cuda")
    m, v = ops.adamw_values(codes, codes, scales)

    def number(c, fraction):
        e, f = c >> fraction, (c & ((1 << fraction) - 1)) / (1 << fraction)
        return (1 + f) * 2.0 ** (e - 16) if e else f * 2.0 ** -15

    for c in range(256):
        want = number(c & 127, 3) / number(127, 3) * 3.0 * (-1 if c >= 128 else 1)
        assert abs(m[c].item() - want) <= 3 * U * abs(want)
        want = (number(c, 4) / number(255, 4) * 0.5) ** 2
        assert abs(v[c].item() - want) <= 7 * U * want
    assert number(127, 3) == 0.9375 and number(255, 4) == 0.96875


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("param", [torch.float32, torch.bfloat16, torch.float16])
def test_moments_in_8_bits(param, shift):
    """Parameters move by the unrounded moments; each moment is one of the two codes beside its value, its block's largest the scale."""
    step, sizes = 2, [1, 255, 256, 257, 4099, 70001]
    g = _random(2)
    params = [(0.1 * torch.randn(n + shift, generator=g)).to(param).cuda()[shift:] for n in sizes]
    grads = [(1e-2 * torch.randn(n + shift, generator=g) * torch.exp(3 * torch.randn(n + shift, generator=g))).to(param).cuda()[shift:] for n in sizes]
    ms, vs, scales = zip(*[_state(n, 8, 3 + n) for n in sizes])
    before = [(p.clone(), *ops.adamw_values(m, v, s)) for p, m, v, s in zip(params, ms, vs, scales)]
    ops.adamw_step(params, grads, ms, vs, scales, step=step, seed=11, **HYPER)
    for p, g, m, v, s, (p0, m0, v0) in zip(params, grads, ms, vs, scales, before):
        p1, m1, v1, rm, rv, rp = _exact(p0, g, m0, v0, step, **HYPER)
        if param != torch.float32:
            rp = rp + torch.finfo(param).eps / 2 * p1.abs() + torch.finfo(param).smallest_normal * torch.finfo(param).eps
        _within(p, p1, rp)
        n = p.numel()
        pad = lambda t: torch.nn.functional.pad(t, (0, -n % 256)).view(-1, 256)  # noqa: E731
        got_m, got_v = (t.double() for t in ops.adamw_values(m, v, s))
        for got, want, room, scale, fraction, top in ((got_m.abs(), m1.abs(), rm, s[:, 0], 3, 0.9375), (got_v.sqrt(), v1.sqrt(), rv / v1.sqrt().clamp(min=1e-30), s[:, 1], 4, 0.96875)):
            _within(scale, pad(want).amax(1), pad(room).amax(1) + 2 * U * scale.double())
            scale = scale.double().repeat_interleave(256)[:n]
            # within a code step, whose size is that of the larger of the two numbers' neighbourhoods; a root above 0 may be raised to the first code
            near = torch.maximum(got, want)
            off = (got - want).abs()
            assert (off <= _step_of_code(near, scale, fraction, top) * (1 + 1e-5) + room + 1e-6 * scale * 2.0 ** -18).all()
        assert (got_v > 0).eq(v1 > 0).all()
        assert ((got_m == 0) | (got_m.sign() == m1.sign())).all()


def _eight(n, seed, steps, gradient, b2=0.999):
    p, m, v, s = torch.zeros(n, device="cuda"), *(torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)), torch.zeros((n + 255) // 256, 2, device="cuda")
    for t in range(1, steps + 1):
        ops.adamw_step([p], [gradient], [m], [v], [s], step=t, seed=seed, lr=1e-3, betas=(0.9, b2))
    return p, m, v, s


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits_and_another_seed_others():
    g = torch.randn(10000, generator=_random(4)).cuda()
    a, b, c = _eight(10000, 1, 4, g), _eight(10000, 1, 4, g), _eight(10000, 2, 4, g)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(a[1], c[1]) and not torch.equal(a[2], c[2])


@pytest.mark.gpu
def test_moments_in_8_bits_follow_what_moves_by_less_than_a_code_step():
    """200 steps of one gradient from v = g^2 / 4 on: v moves by 0.3 % of itself a step at most and its root by 0.15 %, a code step is 3 % and more.  Rounded to nearest it would
    stay where it is.  What the rounding adds: a root r in a code step c <= r / 16 is rounded with a variance of at most c^2 / 4, so v = r^2 gets r^2 / 1024 on average, less than a
    thousandth of itself a step, and keeps it: after 200 steps at most 20 %.  Its noise: 200 (r / 32)^2 is a sigma of 0.44 of r, over 2^16 values with random bits of their own
    0.0017 of the mean."""
    n = 1 << 16
    g = (0.75 + 0.5 * torch.rand(n, generator=_random(5))).cuda() * 1e-3
    p, m, s = torch.zeros(n, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n // 256, 2, device="cuda")
    v = torch.zeros_like(m)
    ops.adamw_step([p], [g], [m], [v], [s], step=1, betas=(0.9, 0.75))  # v = g^2 / 4
    first = ops.adamw_values(m, v, s)[1].double()
    assert abs((first / (g.double().square() / 4)).mean() - 1) <= 0.01
    for t in range(2, 202):
        ops.adamw_step([p], [g], [m], [v], [s], step=t, betas=(0.9, 0.999))
    got_m, got_v = (t.double() for t in ops.adamw_values(m, v, s))
    want = (1 - 0.75 * 0.999 ** 200) * g.double().square()
    ratio = (got_v / want).mean().item()
    assert 1 - 0.01 <= ratio <= 1.22, ratio
    assert want.mean() >= 1.5 * first.mean()
    assert abs((got_m / g.double()).mean().item() - 1) <= 0.01


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_a_launch_takes(bits):
    """1000 tensors, in three launches, each as in a call of its own (with the random bits of its place in the list)."""
    g = _random(6)
    sizes = [int(n) for n in torch.randint(0, 700, (1000,), generator=g)]
    params, grads = [torch.randn(n, generator=g).cuda() for n in sizes], [torch.randn(n, generator=g).cuda() for n in sizes]
    states = [_state(n, bits, 100 + i) for i, n in enumerate(sizes)]
    kept = [(p.clone(), tuple(t.clone() if t is not None else None for t in s)) for p, s in zip(params, states)]
    ms, vs, scales = (list(t) for t in zip(*states))
    ops.adamw_step(params, grads, ms, vs, scales if bits == 8 else None, step=1, **HYPER)
    for i in range(0, 1000, 37):
        p0, (m0, v0, s0) = kept[i]
        if bits == 32:
            ops.adamw_step([p0], [grads[i]], [m0], [v0], step=1, **HYPER)
        else:
            ops.adamw_step([*(torch.zeros(0, device="cuda") for _ in range(i)), p0], [*(torch.zeros(0, device="cuda") for _ in range(i)), grads[i]],
                           [*(torch.zeros(0, device="cuda", dtype=torch.uint8) for _ in range(i)), m0], [*(torch.zeros(0, device="cuda", dtype=torch.uint8) for _ in range(i)), v0],
                           [*(torch.zeros(0, 2, device="cuda") for _ in range(i)), s0], step=1, **HYPER)
            assert torch.equal(scales[i], s0)
        assert torch.equal(params[i], p0) and torch.equal(ms[i], m0) and torch.equal(vs[i], v0)


@pytest.mark.gpu
def test_what_is_not_finite():
    """A NaN stays in its value with 32 bits; with 8 its block of 256 becomes NaN a step later, and the others stay as they were."""
    g = torch.full((600,), 1e-2, device="cuda")
    g[300] = float("nan")
    p, m, v = torch.ones(600, device="cuda"), torch.zeros(600, device="cuda"), torch.zeros(600, device="cuda")
    ops.adamw_step([p], [g], [m], [v], step=1)
    assert all(t.isnan().sum() == 1 and t[300].isnan() for t in (p, m, v))
    for bad in (float("nan"), float("inf"), -float("inf")):
        g[300] = bad
        p, m, v, s = _eight(600, 0, 1, g)
        assert p.isfinite().sum() == 599
        m, v = ops.adamw_values(m, v, s)
        for t in (m, v):
            assert t[256:512].isnan().all() and t[:256].isfinite().all() and t[512:].isfinite().all()
    # nothing at all, and values below what a block holds
    for tiny in (0.0, 1e-35):
        p, m, v, s = _eight(300, 0, 2, torch.full((300,), tiny, device="cuda"))
        assert (s == 0).all() and (m == 0).all() and (v == 0).all() and p.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_orders_of_memory(bits):
    """A parameter that lies transposed, with a gradient that does not, and one whose gradient has gaps."""
    g = _random(7)
    p = torch.randn(40, 70, generator=g).cuda().t()
    grad, wide = torch.randn(70, 40, generator=g).cuda(), torch.randn(33, 64, generator=g).cuda()
    q = torch.randn(33, 32, generator=g).cuda()
    like = torch.uint8 if bits == 8 else torch.float32
    params, grads = [p, q], [grad, wide[:, ::2]]
    ms, vs = [torch.zeros_like(t, dtype=like) for t in params], [torch.zeros_like(t, dtype=like) for t in params]
    scales = [torch.zeros((t.numel() + 255) // 256, 2, device="cuda") for t in params] if bits == 8 else None
    want = [_exact(a, b, torch.zeros_like(b), torch.zeros_like(b), 1, **HYPER) for a, b in zip(params, grads)]
    ops.adamw_step(params, grads, ms, vs, scales, step=1, **HYPER)
    for a, (p1, m1, _, rm, _, rp), m in zip(params, want, ms):
        _within(a, p1, rp)
        if bits == 32:
            _within(m, m1, rm)
    with pytest.raises(ValueError, match="strides"):
        ops.adamw_step([p], [grad], [torch.zeros(70, 40, device="cuda")], [ms[0]] if bits == 32 else [torch.zeros_like(p)], step=1)
    with pytest.raises(ValueError, match="gaps"):
        ops.adamw_step([wide[:, ::2]], [q], [torch.zeros_like(q)], [torch.zeros_like(q)], step=1)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_go_on_counting(bits):
    g = _random(8)
    sizes = [300, 5, 256 * 40]

    def fresh():
        r = _random(9)
        params = [torch.randn(n, generator=r).cuda() for n in sizes]
        like = torch.uint8 if bits == 8 else torch.float32
        return params, [torch.zeros(n, dtype=like, device="cuda") for n in sizes], [torch.zeros(n, dtype=like, device="cuda") for n in sizes], \
            [torch.zeros((n + 255) // 256, 2, device="cuda") for n in sizes] if bits == 8 else None

    grads = [torch.randn(n, generator=g).cuda() for n in sizes]
    params, ms, vs, scales = fresh()
    step, lr = torch.zeros((), dtype=torch.int64, device="cuda"), torch.tensor(2.0 ** -9, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step += 1
        ops.adamw_step(params, grads, ms, vs, scales, step=step, lr=lr, seed=4)
    for _ in range(3):
        graph.replay()
    lr.fill_(2.0 ** -8)
    graph.replay()
    other, om, ov, os_ = fresh()
    for t in range(1, 5):
        ops.adamw_step(other, grads, om, ov, os_, step=t, lr=2.0 ** -9 if t < 4 else 2.0 ** -8, seed=4)
    for a, b in zip(ms + vs, om + ov):
        assert torch.equal(a, b)
    for a, b in zip(params, other):  # the device's powers may be a step of fp32 from the host's, in each of four steps
        assert (a - b).abs().max() <= 4 * 4 * U * (b.abs().max() + 4 * 2.0 ** -8)


@pytest.mark.gpu
def test_two_streams_and_saved_tensors():
    """Steps of two sets of tensors at once; whoever saved a parameter for a backward pass is told that it has changed."""
    g = _random(10)
    a, b = [torch.randn(1 << 20, generator=g).cuda() for _ in range(2)]
    grad = torch.randn(1 << 20, generator=g).cuda()
    want = [_exact(t, grad, torch.zeros_like(t), torch.zeros_like(t), 1, **HYPER) for t in (a, b)]
    state = [torch.zeros_like(a) for _ in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for t, s, k in ((a, streams[0], 0), (b, streams[1], 2)):
        with torch.cuda.stream(s):
            ops.adamw_step([t], [grad], [state[k]], [state[k + 1]], step=1, **HYPER)
    torch.cuda.synchronize()
    for t, w in zip((a, b), want):
        _within(t, w[0], w[5])
    w = torch.ones(4, device="cuda", requires_grad=True)
    x = torch.ones(4, device="cuda", requires_grad=True)
    y = (w * x).sum()
    ops.adamw_step([w], [torch.ones(4, device="cuda")], [torch.zeros(4, device="cuda")], [torch.zeros(4, device="cuda")], step=1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def _args(device="cuda"):
    f = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=device)  # noqa: E731
    return [f(300)], [f(300)], [f(300)], [f(300)]


@pytest.mark.gpu
def test_refusals():
    p, g, m, v = _args()
    byte = [torch.zeros(300, dtype=torch.uint8, device="cuda")]
    scales = [torch.zeros(2, 2, device="cuda")]
    ops.adamw_step([], [], [], [], step=1)
    refused = [
        ((p, [], m, v), dict(step=1), "lengths"), ((p, g, m, v), dict(step=0), "count from 1"), ((p, g, m, v), dict(step=1, betas=(1.0, 0.9)), "betas"),
        ((p, g, m, v), dict(step=1, lr=-1.0), "negative"), ((p, g, m, v), dict(step=1, eps=-1.0), "negative"), ((p, g, m, v, scales), dict(step=1), "type"),
        ((p, g, byte, byte), dict(step=1), "type"), ((p, [g[0][:299]], m, v), dict(step=1), "shape"), ((p, g, [m[0][:299]], v), dict(step=1), "shape"),
        ((p, g, byte, [byte[0].clone()], [torch.zeros(1, 2, device="cuda")]), dict(step=1), "every 256"), ((p, g, m, m), dict(step=1), "overlap"),
        ((p, p, m, v), dict(step=1), "overlap"), ((p * 2, g * 2, m * 2, v * 2), dict(step=1), "overlap"), ((p, [g[0].half()], m, v), dict(step=1, lr=torch.zeros(2, device="cuda")), "one value"),
        (([p[0].half()], g, m, v), dict(step=1), "gradient|grads"), (([p[0].double()], g, m, v), dict(step=1), "float32, bfloat16"), ((p, [g[0].cpu()], m, v), dict(step=1), "CUDA"),
        ((p, g, m, v), dict(step=torch.ones(1, device="cuda")), "one value"), ((p, [g[0].to_sparse()], m, v), dict(step=1), "dense"),
        (([torch._neg_view(p[0])], g, m, v), dict(step=1), "in its memory"),
    ]
    for args, kw, match in refused:
        with pytest.raises((ValueError, NotImplementedError), match=match):
            ops.adamw_step(*args, **kw)
    base = torch.zeros(500, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        ops.adamw_step([base[:300], base[200:]], [g[0], g[0]], [m[0], v[0]], [torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")], step=1)
    ops.adamw_step([base[:300]], [torch._neg_view(g[0])], m, v, step=1)
    with pytest.raises(ValueError):
        ops.adamw_values(m[0], v[0], scales[0])
    with pytest.raises(ValueError, match="every 256"):
        ops.adamw_values(byte[0], byte[0], scales[0][:1])
    assert all((t[0] == 0).all() for t in (p, g, m, v))


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        ops.adamw_step(*_args("cpu"), step=1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.adamw_values(torch.zeros(3, dtype=torch.uint8), torch.zeros(3, dtype=torch.uint8), torch.zeros(1, 2))
    for kw in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(bits=16)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_c_entry_points_refuse():
    """Nothing below is launched."""
    lib = _lib.cuda()

    class Tensor(C.Structure):
        _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("m", C.c_void_p), ("v", C.c_void_p), ("scales", C.c_void_p), ("n", C.c_size_t), ("number", C.c_uint32)]

    good = dict(param=4096, grad=4096, m=4096, v=4096, scales=4096, n=10, number=0)

    def call(entry, pt=0, gt=0, bits=8, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, decay=0.0, step=1, lr_at=None, step_at=None, count=1):
        t = Tensor(**entry)
        return lib.hc_adamw(C.byref(t), count, pt, gt, bits, lr, lr_at, b1, b2, eps, decay, step, step_at, 0, None)

    for bad in (dict(param=4098), dict(grad=4097), dict(scales=4100), dict(param=None), dict(grad=None), dict(m=None), dict(v=None), dict(scales=None), dict(n=1 << 40)):
        assert call({**good, **bad}) == 4, bad
    assert call({**good, "m": 4098}, bits=32) == 4 and call({**good, "v": 4098}, bits=32) == 4
    for bad in (dict(pt=3), dict(gt=-1), dict(pt=1, gt=0), dict(pt=1, gt=2), dict(bits=16), dict(lr=-1.0), dict(lr=float("nan")), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(decay=-1.0),
                dict(step=0), dict(lr_at=4097), dict(step_at=4100)):
        assert call(good, **bad) == 4, bad
    assert lib.hc_adamw(None, 1, 0, 0, 8, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 1, None, 0, None) == 4
    assert lib.hc_adamw(None, 0, 0, 0, 8, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 1, None, 0, None) == 0
    values = dict(m=4096, v=4096, s=4096, n=10, mo=4096, vo=4096)
    for bad in (dict(m=None), dict(s=4100), dict(mo=4098), dict(vo=4097), dict(n=1 << 40)):
        assert lib.hc_adamw_values(*{**values, **bad}.values(), None) == 4
    assert lib.hc_adamw_values(*{**values, "n": 0}.values(), None) == 0


@pytest.mark.gpu
def test_optimiser_against_torch_in_64_bits():
    """Five steps, one parameter without a gradient in the second: each step is off by the step's own rounding and what the steps before have left."""
    g = _random(12)
    shapes = [(33, 17), (5,), (1000,)]
    params = [torch.nn.Parameter(torch.randn(*s, generator=g).cuda()) for s in shapes]
    exact = [torch.nn.Parameter(p.detach().double()) for p in params]
    opt, ref = AdamW(params, **HYPER), torch.optim.AdamW(exact, **HYPER)
    for t in range(5):
        for i, (p, q) in enumerate(zip(params, exact)):
            p.grad = None if t == 1 and i == 1 else torch.randn(*shapes[i], generator=g).cuda()
            q.grad = None if p.grad is None else p.grad.double()
        opt.step()
        ref.step()
    for p, q in zip(params, exact):
        # a step moves a parameter by 10 lr at most; five steps of 4 U of the parameter and 40 U of the movement
        assert (p.double() - q).abs().max() <= 5 * (4 * U * 5.0 + 40 * U * 10 * HYPER["lr"])
        assert opt.state[p]["step"] == int(ref.state[q]["step"])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_optimiser_state_saved_and_loaded(bits, kind):
    g = _random(13)
    start = [torch.randn(300, 7, generator=g).to(kind).cuda(), torch.randn(9, generator=g).to(kind).cuda()]
    grads = [[torch.randn(*p.shape, generator=g).to(kind).cuda() for p in start] for _ in range(4)]

    def steps(opt, params, which):
        for t in which:
            for p, d in zip(params, grads[t]):
                p.grad = d
            opt.step()

    whole = [torch.nn.Parameter(p.clone()) for p in start]
    opt = AdamW(whole, bits=bits, lr=1e-2)
    steps(opt, whole, range(4))
    half = [torch.nn.Parameter(p.clone()) for p in start]
    first = AdamW(half, bits=bits, lr=1e-2)
    steps(first, half, range(2))
    second = AdamW(half)
    second.load_state_dict(copy.deepcopy(first.state_dict()))
    assert second.state[half[0]]["exp_avg"].dtype == (torch.uint8 if bits == 8 else torch.float32)
    steps(second, half, range(2, 4))
    for a, b in zip(whole, half):
        assert torch.equal(a, b) and all(torch.equal(opt.state[a][n], second.state[b][n]) for n in ("exp_avg", "exp_avg_sq"))


@pytest.mark.gpu
def test_optimiser_captured():
    """The group's step is counted on the device; a captured step, replayed, is the next one."""
    g = _random(14)
    p = torch.nn.Parameter(torch.randn(500, generator=g).cuda())
    q = torch.nn.Parameter(p.detach().clone())
    p.grad, q.grad = (t.detach() for t in (torch.randn(500, generator=g).cuda(),) * 2)
    lr = torch.tensor(2.0 ** -7, device="cuda")
    opt, ref = AdamW([p], lr=lr, capturable=True), AdamW([q], lr=2.0 ** -7)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    graph.replay()
    for _ in range(3):
        ref.step()
    assert int(opt.param_groups[0]["steps"]) == 3
    assert (p - q).abs().max() <= 3 * 4 * U * (q.abs().max() + 1)
    again = AdamW([torch.nn.Parameter(p.detach().clone())], capturable=True)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert int(again.param_groups[0]["steps"]) == 3


@pytest.mark.gpu
def test_muon_with_this_adamw():
    cfg = GPT2Config.tiny()
    cfg.fused = True
    torch.manual_seed(0)
    model = GPT2(cfg).cuda()
    tok = torch.randint(0, 257, (2, 33), generator=_random(15)).cuda()
    opt = muon_with_adamw(model, adam_bits=8)
    assert isinstance(opt.optimizers[1], AdamW) and opt.optimizers[1].param_groups[0]["bits"] == 8
    for _ in range(2):
        opt.zero_grad()
        model(tok[:, :-1], tok[:, 1:]).backward()
        opt.step()
    assert all(p.isfinite().all() for p in model.parameters())


def _trainer(rank, world, bits):
    from tirocinio_triennale_b200.models import train_dp

    args = argparse.Namespace(model="tiny", steps=3, warmup=1, batch=2, seq=32, eb=1e-6, lr=1e-3, bucket_mb=0.05, cpu=False, save=None, resume=None, save_compressed_eb=0.0, fused=True,
                              optimizer="adamw", muon_lr=0.02, adam_bits=bits)
    out = train_dp.run(args, True, rank, world, torch.device("cuda", 0))
    assert out["steps_done"] == 4 and out["last_loss_rank0"] == out["last_loss_rank0"]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_trainer_with_this_adamw(bits):
    run_ranks(_trainer, 1, backend="nccl", args=(bits,))
