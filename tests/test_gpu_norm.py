"""Layer norm and its gradients against the formulas in 64 bits.

Tolerances count roundings.  u is half a step of fp32.  A sum of a row goes through at most 64 additions in a line (8 a
group and thread, shuffles, warps), so it is off by at most 64 u times the sum of absolute values; a sum over rows through at
most rows + 64.  The result's own rounding is half a step of its type."""
import ctypes as C

import pytest
import torch

from tirocinio_triennale_b200 import _lib, ops

U = torch.finfo(torch.float32).eps / 2
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half_step(t):
    return torch.finfo(t).eps / 2


def make(rows, width, kind, seed=0, param=F32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * 2 + torch.randn(width, generator=g)
    return x.to(kind).cuda(), (1 + 0.3 * torch.randn(width, generator=g)).to(param).cuda(), torch.randn(width, generator=g).to(param).cuda(), g


def check(x, w, b, dy, out, eps=1e-5):
    """Runs forward and backward and compares everything."""
    rows, width = x.numel() // x.shape[-1], x.shape[-1]
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = ops.layer_norm(*leaves, eps=eps, out_dtype=out)
    have = [t for t in leaves if t is not None]
    grads = dict(zip([i for i, t in enumerate(leaves) if t is not None], torch.autograd.grad(y, have, dy)))
    assert y.dtype == out and y.shape == x.shape and torch.equal(y, ops.layer_norm(x, w, b, eps=eps, out_dtype=out))
    X, D = x.double().reshape(rows, width), dy.double().reshape(rows, width)
    W = torch.ones(width, device="cuda", dtype=torch.float64) if w is None else w.double()
    B = torch.zeros_like(W) if b is None else b.double()
    mean, r = X.mean(1, keepdim=True), (X.var(1, unbiased=False, keepdim=True) + eps).rsqrt()
    h = (X - mean) * r
    dh = 64 * U * X.abs().mean(1, keepdim=True) * r + 44 * U * h.abs()  # how far a normalised value is off
    want = h * W + B
    tol = half_step(out) * want.abs() + 1.01 * (W.abs() * dh + 2 * U * (want.abs() + B.abs())) + 1e-37
    assert ((y.double().reshape(rows, width) - want).abs() <= tol).all()
    g = D * W
    along, flat = (g * h).mean(1, keepdim=True), g.mean(1, keepdim=True)
    want = r * (g - flat - h * along)
    size = g.abs() + g.abs().mean(1, keepdim=True) + h.abs() * (g * h).abs().mean(1, keepdim=True)
    tol = half_step(x.dtype) * want.abs() + 1.01 * r * (110 * U * size + dh * (g * h).abs().mean(1, keepdim=True) + h.abs() * (g.abs() * dh).mean(1, keepdim=True)) + 1e-37
    if x.dtype == F16:
        tol = tol + 2.0 ** -25
    assert ((grads[0].double().reshape(rows, width) - want).abs() <= tol).all()
    for i, value, size in ((1, D * h, (D * h).abs() * (rows + 64) * U + D.abs() * dh), (2, D, D.abs() * (rows + 64) * U)):
        if i in grads:
            want = value.sum(0)
            t = (w if i == 1 else b).dtype
            assert grads[i].dtype == t
            assert ((grads[i].double() - want).abs() <= half_step(t) * want.abs() + 1.01 * size.sum(0) + 1e-30).all()


WIDTHS = [1, 2, 7, 8, 31, 64, 255, 256, 257, 768, 1000, 1016, 1017, 1024, 1025, 2040, 2048, 2049, 4088, 4095, 4096, 5003, 8184, 8185, 8192, 8193, 20001]


@pytest.mark.gpu
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("kind,out", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16)])
def test_widths(width, kind, out):
    x, w, b, g = make(37, width, kind, width)
    check(x, w, b, torch.randn(37, width, generator=g).to(out).cuda(), out)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,out", [(F32, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("width", [768, 773, 9001])
def test_other_types(kind, out, width):
    x, w, b, g = make(19, width, kind, 1, BF16)
    check(x, w, b, torch.randn(19, width, generator=g).to(out).cuda(), out)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 300, 5000])
@pytest.mark.parametrize("width", [64, 771, 4100])
def test_rows(rows, width):
    x, w, b, g = make(rows, width, BF16, rows)
    check(x, w, b, torch.randn(rows, width, generator=g).to(BF16).cuda(), BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("has_weight,has_bias", [(False, False), (True, False), (False, True)])
def test_without_scale_or_shift(has_weight, has_bias):
    x, w, b, g = make(50, 384, F32, 3)
    check(x, w if has_weight else None, b if has_bias else None, torch.randn(50, 384, generator=g).cuda(), F32)


@pytest.mark.gpu
def test_far_offset_and_constant_rows():
    x, w, b, g = make(64, 768, F32, 4)
    x += 1000.0
    check(x, w, b, torch.randn(64, 768, generator=g).cuda(), F32)
    x = torch.full((3, 500), 5.0, device="cuda")
    y = ops.layer_norm(x)
    assert torch.equal(y, torch.zeros_like(y))


@pytest.mark.gpu
def test_views_and_gradients_with_gaps():
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(3, 41, 1000, generator=g).cuda()
    w, b = torch.randn(500, generator=g).cuda(), torch.randn(500, generator=g).cuda()
    for x in (wide[..., ::2], wide[..., 1:501], wide.transpose(0, 1)[..., :500], torch.randn(20 * 500 + 1, generator=g).cuda()[1:].view(20, 500)):
        check(x, w, b, torch.randn(*x.shape, generator=g).cuda(), F32)
    x = torch.randn(40, 500, generator=g).cuda().requires_grad_()
    (dx,) = torch.autograd.grad(ops.layer_norm(x, w, b).sum(), (x,))  # the gradient of a sum has strides of 0
    assert dx.shape == x.shape and torch.isfinite(dx).all()


@pytest.mark.gpu
def test_gradient_against_differences():
    x, w, b, g = make(3, 96, F32, 6)
    dy = torch.randn(3, 96, generator=g).cuda()
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)

    def f(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return ((c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * w + b) * dy.double()).sum()

    base = [t.double() for t in (x, w, b)]
    for k in range(3):
        for at in ((0,), (17,), (95,)):
            at = (1, *at) if k == 0 else at
            ends = []
            for s in (1e-4, -1e-4):
                moved = [t.clone() for t in base]
                moved[k][at] += s
                ends.append(f(*moved))
            # differences of step 1e-4 are off by the third derivative / 6 * 1e-8; every derivative here is below 1e3
            assert abs((ends[0] - ends[1]) / 2e-4 - grads[k][at].double()) <= 2e-6 + 1e-4 * abs(grads[k][at].double())


@pytest.mark.gpu
def test_empty_and_partial_gradients():
    w, b = torch.ones(64, device="cuda", requires_grad=True), torch.zeros(64, device="cuda", requires_grad=True)
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()
    x, w, b, g = make(33, 200, F32, 7)
    dy = torch.randn(33, 200, generator=g).cuda()
    all_three = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(ops.layer_norm(*all_three), all_three, dy)
    for k in range(3):
        one = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(ops.layer_norm(*one), (one[k],), dy)[0], want[k])


@pytest.mark.gpu
def test_same_bits_every_time_other_streams_and_graphs():
    x, w, b, g = make(3000, 776, BF16, 8)
    dy = torch.randn(3000, 776, generator=g).to(BF16).cuda()

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = ops.layer_norm(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))

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
    dy.copy_(dy.flip(0))
    other = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, there))
    assert all(torch.equal(p, q) for p, q in zip(other, caught))


@pytest.mark.gpu
def test_refusals():
    x = torch.randn(4, 16, device="cuda")
    w = torch.ones(16, device="cuda")
    for bad in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x.cpu()), lambda: ops.layer_norm(x, w[:8]),
                lambda: ops.layer_norm(x, w, w.half()), lambda: ops.layer_norm(x, w.cpu()), lambda: ops.layer_norm(x, eps=-1.0),
                lambda: ops.layer_norm(x, eps=float("nan")), lambda: ops.layer_norm(x.half(), out_dtype=BF16),
                lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(x, out_dtype=torch.int32), lambda: ops.layer_norm(x, w[None])):
        with pytest.raises(ValueError):
            bad()


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        ops.layer_norm(torch.ones(2, 8))
    lib = _lib.cuda()
    p = C.c_void_p(4096)  # never read: every call below is refused before anything is launched
    good = dict(x=p, xt=0, w=None, b=None, pt=0, y=p, yt=0, st=None, rows=4, width=16, eps=1e-5)

    def forward(**kw):
        return lib.hc_layer_norm(*{**good, **kw}.values(), None)

    for kw in (dict(xt=3), dict(yt=-1), dict(pt=9), dict(xt=1, yt=2), dict(width=0), dict(width=1 << 31), dict(rows=1 << 50), dict(eps=-1.0),
               dict(x=C.c_void_p(4104)), dict(y=C.c_void_p(4098)), dict(x=None), dict(y=None)):
        assert forward(**kw) == 4, kw
    assert forward(rows=0) == 0
    back = lambda dw, db, dx=p, s=p, n=1 << 30: lib.hc_layer_norm_backward(p, 0, p, 0, None, 0, p, dx, dw, db, 4, 16, s, n, None)  # noqa: E731
    assert back(p, None) == 4 and back(None, p) == 4 and back(p, p, s=None) == 4 and back(p, p, n=8) == 4 and back(None, None, C.c_void_p(4100)) == 4
    assert back(None, None, None) == 0


def test_sizes_that_wrap_are_refused():
    """rows x width beyond 2^60 is refused also where 64 bits count it from 0 again."""
    lib = _lib.cuda()
    p = C.c_void_p(4096)  # never read: every call below is refused before anything is launched
    for rows, width in ((1 << 40, 1 << 24), (1 << 40, 1 << 30), (1 << 39, (1 << 25) + 8), (1 << 37, 1 << 27)):
        assert lib.hc_layer_norm(p, 0, None, None, 0, p, 0, None, rows, width, 1e-5, None) == 4
        assert lib.hc_layer_norm_backward(p, 0, p, 0, None, 0, p, p, None, None, rows, width, None, 0, None) == 4
