"""Products with bias, activation and residual, and their gradients, against the formulas in 64 bits.

Tolerances count roundings.  u and h are half a step of fp32 and of the operands' type.  Products of 16-bit numbers are exact in
fp32; a sum over k of them goes through at most k / 16 + 20 additions in a line, each off by at most a whole step (the tensor core
need not round to nearest).  An activation's slope is at most 1.13, the slope's own slope at most 0.8 (ReLU apart).  Gradients see
the argument of the activation rounded to the operands' type, and are themselves rounded to it before the products."""
import ctypes as C

import pytest
import torch
import torch.nn.functional as F

from tirocinio_triennale_b200 import _lib, ops

U = torch.finfo(torch.float32).eps / 2
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ACT = {None: lambda z: z, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "relu": F.relu, "silu": F.silu}


def half_step(t):
    return torch.finfo(t).eps / 2


def least(t):
    return 2.0 ** -25 if t == F16 else 1e-37  # half of the smallest number apart from 0


def sums(k):
    return (k / 16 + 20) * 2 * U


def make(m, k, n, kind, seed=0, bias=F32, residual=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(kind).cuda()
    w = (torch.randn(n, k, generator=g) / k ** 0.5).to(kind).cuda()
    b = None if bias is None else torch.randn(n, generator=g).to(bias).cuda()
    r = None if residual is None else torch.randn(m, n, generator=g).to(residual).cuda()
    dy = torch.randn(m, n, generator=g).to(kind if r is None else residual).cuda()
    return x, w, b, r, dy


def check(x, w, b, r, dy, act=None, out_dtype=None):
    t = x.dtype
    leaves = [None if v is None else v.detach().requires_grad_() for v in (x, w, b, r)]
    y = ops.linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3], out_dtype=out_dtype)
    assert y.dtype == (r.dtype if r is not None else out_dtype or t) and y.shape == (*x.shape[:-1], w.shape[0])
    assert torch.equal(y, ops.linear(x, w, b, activation=act, residual=r, out_dtype=out_dtype))
    have = [i for i, v in enumerate(leaves) if v is not None]
    grads = dict(zip(have, torch.autograd.grad(y, [leaves[i] for i in have], dy)))
    m, k, n = x.numel() // x.shape[-1], x.shape[-1], w.shape[0]
    X, W, D = x.double().reshape(m, k), w.double(), dy.double().reshape(m, n)
    z = X @ W.t()
    ez = sums(k) * (X.abs() @ W.abs().t())
    if b is not None:
        z = z + b.double()
        ez = ez + U * z.abs()
    z = z.requires_grad_()
    a = ACT[act](z)
    (slope,) = torch.autograd.grad(a.sum(), (z,))
    a, z = a.detach(), z.detach()
    want = a if r is None else a + r.double().reshape(m, n)
    h = half_step(y.dtype)
    room = 1.01 * (h * want.abs() + 1.13 * ez + 8 * U * (a.abs() + want.abs())) + least(y.dtype)
    assert ((y.double().reshape(m, n) - want).abs() <= room).all()
    h = half_step(t)
    dz = D * slope
    if act is None:
        e = torch.zeros_like(dz)
    else:
        move = h * z.abs() + ez + least(t)
        e = D.abs() * (0.8 * move + 8 * U)
        if act == "relu":
            e = torch.where(z.abs() <= move, D.abs(), 0.0)
    if 2 in grads:
        want = dz.sum(0)
        assert grads[2].dtype == b.dtype
        assert ((grads[2].double() - want).abs() <= 1.01 * (e.sum(0) + (m + 64) * U * (dz.abs() + e).sum(0) + half_step(b.dtype) * want.abs()) + least(b.dtype)).all()
    if 3 in grads:
        assert torch.equal(grads[3], dy)
    e = e + h * dz.abs() + least(t)
    for i, left, right, el in ((0, dz, W, e), (1, dz.t(), X, e.t())):
        want = left @ right
        room = el @ right.abs() + sums(left.shape[1]) * ((left.abs() + el) @ right.abs()) + h * want.abs() + least(t)
        got = grads[i]
        assert got.dtype == t and got.shape == (x, w)[i].shape
        assert ((got.double().reshape(want.shape) - want).abs() <= 1.01 * room).all()


SIZES = [(9, 8, 8), (16, 64, 64), (100, 72, 136), (128, 128, 256), (129, 130, 131), (200, 7, 1), (300, 1, 300), (130, 96, 257), (257, 1000, 520), (1000, 200, 2304), (640, 2048, 384), (64, 4096, 64), (8200, 104, 312), (5003, 33, 77)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("kind", [BF16, F16])
def test_sizes(m, k, n, kind):
    check(*make(m, k, n, kind, m))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [*range(1, 10), 15, 16, 17, 33])
@pytest.mark.parametrize("k,n", [(768, 2304), (64, 17), (1001, 33), (5000, 100)])
def test_few_rows(m, k, n):
    check(*make(m, k, n, BF16, m, BF16, F32 if m % 2 else None))
    check(*make(m, k, n, BF16, m, BF16, None if m % 2 else BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu_tanh", "relu", "silu"])
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("m,k,n", [(5, 96, 50), (300, 264, 200), (77, 65, 129)])
def test_activations(act, kind, m, k, n):
    check(*make(m, k, n, kind, 1, kind), act)


@pytest.mark.gpu
@pytest.mark.parametrize("residual", [F32, BF16])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", [(3, 64, 96), (130, 128, 100), (260, 64, 512), (50, 70, 33)])
def test_residuals(residual, act, m, k, n):
    check(*make(m, k, n, BF16, 2, None, residual), act)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,act,residual", [(BF16, None, F32), (F16, "gelu_tanh", None), (BF16, "silu", BF16), (BF16, "relu", None)])
@pytest.mark.parametrize("m,k,n", [(33, 5000, 136), (130, 4104, 1000), (40, 3001, 77), (35, 8192, 8), (300, 6144, 200)])
def test_long_sums_of_few_tiles(m, k, n, kind, act, residual):
    """Sums that are shared out over the GPU, in either direction, with all that follows a product."""
    assert _lib.cuda().hc_linear_bytes(m, k, n) > 0
    check(*make(m, k, n, kind, m + n, kind, residual), act)
    x, w, b, r, dy = make(m, n, k, kind, m, kind, residual)
    check(x, w, b, r, dy, act)


@pytest.mark.gpu
def test_fp32_results():
    x, w, b, _, dy = make(140, 192, 72, BF16, 3)
    check(x, w, b, None, dy.float(), None, F32)
    check(x, w, b, None, dy.float(), "silu", F32)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(150, 70, 90), (513, 200, 700), (1030, 65, 258), (4, 300, 40), (2000, 130, 520)])
@pytest.mark.parametrize("kind", [BF16, F16])
def test_whole_numbers_are_exact(m, k, n, kind):
    """Small whole numbers: every sum is one that each type holds, so each element has one right value."""
    g = torch.Generator().manual_seed(m)
    some = lambda *s: (torch.randint(-1, 2, s, generator=g) * (torch.rand(*s, generator=g) < 0.2)).to(kind).cuda()  # noqa: E731
    x, w, dy = some(m, k), some(n, k), some(m, n)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    y = ops.linear(*leaves)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    for got, want in ((y, x.double() @ w.double().t()), (dx, dy.double() @ w.double()), (dw, dy.double().t() @ x.double())):
        assert want.abs().max() <= 256 and torch.equal(got.double(), want)


@pytest.mark.gpu
def test_views_batches_and_gradients_with_gaps():
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(3, 50, 400, generator=g).to(BF16).cuda()
    w = torch.randn(120, 300, generator=g).to(BF16).cuda() / 17
    for x in (wide[..., :300], wide[..., 1:301], wide[..., ::2][..., :100].repeat(1, 1, 3), wide[:, :, :300].transpose(0, 1), wide[:1, :1, 3:303], wide[:, :2, 3:303]):
        for weight in (w, w.t().contiguous().t(), torch.cat([w, w], 1)[:, 7:307]):
            dy = torch.randn(*x.shape[:-1], 120, generator=g).to(BF16).cuda()
            check(x, weight, None, None, dy)
    x = wide[0, :, :300].detach().requires_grad_()
    (dx,) = torch.autograd.grad(ops.linear(x, w).sum(), (x,))  # the gradient of a sum has strides of 0
    want = w.double().sum(0)
    assert ((dx.double() - want).abs() <= half_step(BF16) * want.abs() + sums(120) * w.double().abs().sum(0)).all()
    out = ops.linear(wide[0, :, :300], w, residual=torch.randn(50, 240, generator=g).cuda()[:, ::2])
    assert out.shape == (50, 120) and out.dtype == F32
    odd = ops.linear(wide[0, :, :300], w[:113])
    assert odd.shape == (50, 113) and odd.stride(0) % 8 == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,stride,first", [(1, 1, 1, 0), (3, 7, 9, 1), (40, 65, 65, 3), (300, 1001, 1003, 5), (64, 96, 104, 0), (17, 8, 11, 2), (5, 4099, 4099, 7)])
def test_rows_that_begin_anywhere(rows, width, stride, first):
    """Copied whole, with zeros up to the next eight, and nothing behind those."""
    src = torch.randint(-1000, 1000, (first + rows * stride,), dtype=torch.int16, device="cuda")
    taken = src[first:].as_strided((rows, width), (stride, 1))
    up = (width + 7) // 8 * 8
    out = torch.full((rows + 1, up + 8), 77, dtype=torch.int16, device="cuda")
    assert _lib.cuda().hc_align_rows(taken.data_ptr(), stride, rows, width, out.data_ptr(), up + 8, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out[:rows, :width], taken) and (out[:rows, width:up] == 0).all() and (out[:, up:] == 77).all() and (out[rows] == 77).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(6,), (1,), (2, 3), ()])
@pytest.mark.parametrize("n", [24, 33])
def test_results_can_be_changed_in_place(shape, n):
    x, w, b, _, _ = make(6, 40, n, BF16)
    x = (x[0] if shape == () else x[:1] if shape == (1,) else x.reshape(*shape, 40)).requires_grad_()
    y = ops.linear(x, w, b)
    assert y.shape == (*shape, n)
    before = y.detach().clone()
    y.mul_(2.0)
    y.sum().backward()
    assert torch.equal(y.detach(), before * 2)
    twice = torch.autograd.grad(ops.linear(x, w, b), x, torch.full_like(before, 2.0))[0]
    assert torch.equal(x.grad, twice)


@pytest.mark.gpu
def test_long_sums_in_parts_with_fp32_results():
    assert _lib.cuda().hc_linear_bytes(64, 8192, 4096) > 0
    check(*make(64, 8192, 4096, BF16, 9, BF16, F32))


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(5, 512, 96), (16, 1001, 50), (64, 8192, 200), (300, 256, 130)])
def test_a_row_of_nan_and_infinities_keeps_to_itself(m, k, n):
    x, w, b, _, _ = make(m, k, n, BF16, 4)
    clean = ops.linear(x, w, b, activation="silu")
    bad = x.clone()
    bad[1, 3], bad[2, 5] = float("nan"), float("inf")
    out = ops.linear(bad, w, b, activation="silu")
    assert out[1].isnan().all() and not out[2].isfinite().all()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.gpu
def test_shared_sums_captured_and_on_two_streams():
    """Each call has its own parts of a sum: two graphs and two streams at once give what one call gives."""
    cases = [make(64, 8192, 256, BF16, 7), make(48, 6144, 512, BF16, 8)]
    want = [ops.linear(x, w, b) for x, w, b, _, _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (x, w, b, _, _), side in zip(cases, streams):
            with torch.cuda.stream(side):
                got.append(ops.linear(x, w, b))
        torch.cuda.synchronize()
        assert all(torch.equal(g, y) for g, y in zip(got, want))
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()
    for x, w, b, _, _ in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(ops.linear(x, w, b))
        graphs.append(graph)
    for _ in range(2):
        for (x, w, b, _, _), graph, out in zip(cases, graphs, outs):
            x.neg_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ops.linear(x, w, b))


@pytest.mark.gpu
def test_rows_of_another_tensor_stay():
    """Tiles that reach over the last row and column store nothing there."""
    x, w, b, _, _ = make(130, 64, 100, BF16, 5)
    lib = _lib.cuda()
    for n, stride in ((100, 112), (99, 101)):
        out = torch.full((133, stride), 7.0, dtype=BF16, device="cuda")
        assert lib.hc_linear(x.data_ptr(), 64, w.data_ptr(), 64, 1, b.data_ptr(), 0, None, 0, out.data_ptr(), 1, stride, None, 0, 0, 130, 64, n, None, 0,
                             torch.cuda.current_stream().cuda_stream) == 0
        assert (out[130:] == 7).all() and (out[:, n:] == 7).all()
        assert torch.equal(out[:130, :n], ops.linear(x, w[:n], b[:n]))


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(150, 100, 99), (40, 65, 257), (3, 100, 30), (300, 7, 9)])
def test_what_lies_between_rows_is_not_read(m, k, n):
    x, w, b, _, dy = make(m, k, n, BF16, 10, None)

    def apart(t):
        wide = torch.full((t.shape[0], (t.shape[1] + 8) // 8 * 8), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, :t.shape[1]] = t
        return wide[:, :t.shape[1]]

    leaves = [apart(x).requires_grad_(), apart(w).requires_grad_()]
    y = ops.linear(*leaves, activation="silu")
    got = (y, *torch.autograd.grad(y, leaves, apart(dy)))
    leaves = [x.requires_grad_(), w.requires_grad_()]
    y = ops.linear(*leaves, activation="silu")
    assert all(torch.equal(p, q) for p, q in zip(got, (y, *torch.autograd.grad(y, leaves, dy))))
    assert all(torch.isfinite(t).all() for t in got)
    y = ops.linear(apart(x.detach()), apart(w.detach()).requires_grad_())
    (dw,) = torch.autograd.grad(y, (y.grad_fn.next_functions[1][0].variable,), apart(dy))  # dy goes into the products as it is
    assert torch.isfinite(dw).all()


@pytest.mark.gpu
def test_partial_gradients_and_no_rows():
    x, w, b, r, dy = make(60, 80, 48, BF16, 6, F32, F32)
    leaves = [v.detach().requires_grad_() for v in (x, w, b, r)]
    want = torch.autograd.grad(ops.linear(*leaves[:3], activation="silu", residual=leaves[3]), leaves, dy)
    for k in range(4):
        one = [v.detach().requires_grad_(i == k) for i, v in enumerate((x, w, b, r))]
        got = torch.autograd.grad(ops.linear(*one[:3], activation="silu", residual=one[3]), (one[k],), dy)
        assert torch.equal(got[0], want[k])
    leaves = [x[:0].detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()]
    y = ops.linear(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy[:0].to(BF16))
    assert y.shape == (0, 48) and dx.shape == (0, 80) and not dw.any() and not db.any()


@pytest.mark.gpu
def test_gradient_against_differences():
    x, w, b, _, dy = make(12, 40, 24, F16, 7)
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    grads = torch.autograd.grad(ops.linear(*leaves, activation="gelu_tanh"), leaves, dy)
    base = [v.double() for v in (x, w, b)]

    def f(x, w, b):
        return (F.gelu(x @ w.t() + b, approximate="tanh") * dy.double()).sum()

    for k, at in ((0, (3, 5)), (0, (11, 39)), (1, (0, 0)), (1, (23, 7)), (2, (9,))):
        ends = []
        for s in (1e-4, -1e-4):
            moved = [v.clone() for v in base]
            moved[k][at] += s
            ends.append(f(*moved))
        # fp16: half a step 5e-4 of each of at most 40 terms of size 1 to 4, and of the result
        assert abs((ends[0] - ends[1]) / 2e-4 - grads[k][at].double()) <= 0.03


@pytest.mark.gpu
def test_infinities_and_nan_stay_in_their_rows():
    x, w, b, _, dy = make(200, 64, 96, BF16, 8)
    x[5, 3], x[150, 60] = float("nan"), float("inf")
    y = ops.linear(x, w, b)
    bad = ~torch.isfinite(y).all(1)
    assert bad.nonzero().flatten().tolist() == [5, 150] and torch.isnan(y[5]).all()
    big = torch.tensor([[3e38], [-3e38], [0.0], [float("nan")]], device="cuda").to(BF16).expand(4, 16).contiguous()
    one = torch.zeros(8, 16, device="cuda", dtype=BF16)
    one[:, 0] = 1
    for act in ("gelu_tanh", "silu", "relu"):
        for rows in (4, 12):  # both kernels
            v = big.repeat(rows // 4, 1).detach().requires_grad_()
            y = ops.linear(v, one, activation=act)
            (d,) = torch.autograd.grad(y, (v,), torch.ones_like(y))
            # sigmoid is held at 2^-60 from there on: the functions stay within 41.5 * 2^-60 < 4e-17 of 0, their slopes (below
            # 41.5 * 2^-60 * 41.5, eight of which are added) within 2e-14
            assert (y[0] == big[0, 0]).all() and (y[1].abs() < 4e-17).all() and (y[2] == 0).all() and torch.isnan(y[3]).all()
            assert float(d[0, 0]) == 8 and abs(float(d[1, 0])) < 2e-14 and float(d[2, 0]) == (0 if act == "relu" else 4) and torch.isnan(d[3, 0])


@pytest.mark.gpu
def test_same_bits_every_time_other_streams_and_graphs():
    x, w, b, r, dy = make(700, 520, 328, BF16, 9, F32, F32)

    def step():
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        y = ops.linear(*leaves, activation="gelu_tanh", residual=r)
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
    other = step()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, there))
    assert all(torch.equal(p, q) for p, q in zip(other, caught))
    assert ops.train_status() == 0


@pytest.mark.gpu
def test_refusals():
    x, w = torch.zeros(4, 16, device="cuda", dtype=BF16), torch.zeros(8, 16, device="cuda", dtype=BF16)
    for bad in (lambda: ops.linear(x.float(), w.float()), lambda: ops.linear(x, w.half()), lambda: ops.linear(x, w[:, :8]), lambda: ops.linear(x, w[0]),
                lambda: ops.linear(x.cpu(), w), lambda: ops.linear(x, w, w[0]), lambda: ops.linear(x, w, activation="tanh"), lambda: ops.linear(x, w, residual=x),
                lambda: ops.linear(x, w, residual=torch.zeros(4, 8, device="cuda", dtype=F16)), lambda: ops.linear(x, w, out_dtype=F16), lambda: ops.linear(x[:, :0], w[:, :0]),
                lambda: ops.linear(x, w, residual=torch.zeros(4, 8, device="cuda"), out_dtype=BF16), lambda: ops.linear(x, w, torch.zeros(8))):
        with pytest.raises(ValueError):
            bad()


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear(torch.ones(2, 8, dtype=BF16), torch.ones(3, 8, dtype=BF16))
    lib = _lib.cuda()
    p = C.c_void_p(4096)  # never read: every call below is refused before anything is launched
    good = dict(x=p, xs=16, w=p, ws=16, type=1, b=None, bt=0, r=None, rs=0, out=p, ot=1, os=24, z=None, zs=0, act=0, m=32, k=16, n=24, scratch=None, bytes=0)

    def forward(**kw):
        return lib.hc_linear(*{**good, **kw}.values(), None)

    for kw in (dict(type=0), dict(type=3), dict(ot=2), dict(bt=3), dict(act=4), dict(act=-1), dict(k=0), dict(n=0), dict(m=1 << 26), dict(xs=15), dict(ws=8), dict(os=23),
               dict(r=p, rs=23), dict(z=p, zs=1), dict(x=None), dict(w=None), dict(out=None), dict(x=C.c_void_p(4098)), dict(xs=17), dict(ws=20), dict(w=C.c_void_p(4104))):
        assert forward(**kw) == 4, kw
    assert forward(m=0) == 0
    long = dict(m=64, k=16384, xs=16384, ws=16384)
    assert lib.hc_linear_bytes(64, 16384, 24) > 4096 and lib.hc_linear_bytes(16, 16384, 24) == 0
    for kw in (dict(), dict(scratch=p, bytes=4096), dict(scratch=C.c_void_p(4104), bytes=1 << 30)):
        assert forward(**long, **kw) == 4, kw
    for kw in (dict(fs=15), dict(ts=15), dict(ts=20), dict(m=1 << 26), dict(k=1 << 26), dict(f=None), dict(t=None), dict(f=C.c_void_p(4097)), dict(t=C.c_void_p(4104))):
        assert lib.hc_align_rows(*{**dict(f=p, fs=17, m=3, k=16, t=p, ts=16), **kw}.values(), None) == 4, kw
    assert lib.hc_align_rows(p, 17, 0, 16, p, 16, None) == 0
    good = dict(dy=p, dt=1, ds=24, z=p, zs=24, act=0, keep=1, x=p, xs=16, w=p, ws=16, type=1, dx=p, dxs=16, dw=p, dws=16, db=p, bt=0, m=32, k=16, n=24,
                scratch=p, bytes=1 << 30)

    def backward(**kw):
        return lib.hc_linear_backward(*{**good, **kw}.values(), None)

    odd = C.c_void_p(4104)
    for kw in (dict(type=0), dict(dt=2), dict(bt=3), dict(act=4), dict(act=-1), dict(ds=23), dict(act=1, zs=23), dict(act=1, z=None), dict(act=1, keep=0), dict(dt=0, keep=0), dict(dy=None),
               dict(xs=15), dict(ws=15), dict(dxs=8), dict(dws=8), dict(x=None), dict(w=None), dict(x=odd), dict(w=odd), dict(xs=17), dict(ws=20), dict(keep=0, dy=odd),
               dict(keep=0, ds=25), dict(scratch=None), dict(scratch=odd), dict(bytes=8), dict(k=0), dict(n=0), dict(m=1 << 26)):
        assert backward(**kw) == 4, kw
    assert backward(dx=None, dw=None, db=None) == 0
    assert lib.hc_linear_backward_bytes(0, 16, 24, 1) == 0


def _columns_apart(m, k, n, act, out_dtype, spoil):
    """What a call gives in all columns but one, with that one spoilt and without."""
    x, w, b, _, _ = make(m, k, n, BF16, 11)
    dy = torch.randn(m, n, generator=torch.Generator().manual_seed(12)).to(out_dtype or BF16).cuda()
    at = 5
    keep = [i for i in range(n) if i != at]

    def step():
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        y = ops.linear(*leaves, activation=act, out_dtype=out_dtype)
        _, dw, db = torch.autograd.grad(y, leaves, dy)
        return y.detach()[:, keep], dw[keep], db[keep], y.detach()[:, at]

    clean = step()
    spoil(w, b, at)
    return clean, step()


@pytest.mark.gpu
@pytest.mark.parametrize("act", [None, "gelu_tanh", "silu", "relu"])
@pytest.mark.parametrize("m,k,n", [(16, 96, 50), (17, 96, 50), (300, 264, 200), (64, 8192, 200), (1000, 64, 512)])
@pytest.mark.parametrize("out_dtype", [None, F32])
def test_a_column_of_nan_keeps_to_itself(m, k, n, act, out_dtype):
    """A bad output unit (NaN in its bias or in its weights) is that unit's alone: every other column of the result, row of
    the weights' gradient and element of the bias's has the bits that it has without it."""

    def bias(w, b, at):
        b[at] = float("nan")

    def weight(w, b, at):
        w[at, 3] = float("nan")

    def infinite(w, b, at):
        w[at] = 0  # inf - inf in every row
        w[at, :2] = torch.tensor([float("inf"), -float("inf")])

    for spoil in (bias, weight, infinite):
        clean, got = _columns_apart(m, k, n, act, out_dtype, spoil)
        assert not torch.isfinite(got[3]).all() and (spoil is infinite or torch.isnan(got[3]).all())
        assert all(torch.isfinite(c).all() and torch.equal(c, g) for c, g in zip(clean[:3], got[:3]))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu_tanh", "silu"])
@pytest.mark.parametrize("out_dtype", [None, F32])
def test_a_value_does_not_depend_on_its_neighbour(act, out_dtype):
    """Columns of which each second one is changed: the others keep their bits, as does their gradient."""
    x, w, b, _, _ = make(300, 264, 200, BF16, 13)
    dy = torch.randn(300, 200, generator=torch.Generator().manual_seed(14)).to(out_dtype or BF16).cuda()

    def step(w, b):
        leaves = [v.detach().requires_grad_() for v in (x, w, b)]
        y = ops.linear(*leaves, activation=act, out_dtype=out_dtype)
        _, dw, db = torch.autograd.grad(y, leaves, dy)
        return y.detach()[:, ::2], dw[::2], db[::2]

    want = step(w, b)
    w[1::2] *= 3
    b[1::2] -= 2
    assert all(torch.equal(p, q) for p, q in zip(want, step(w, b)))


@pytest.mark.gpu
@pytest.mark.parametrize("side", ["rows", "inner"])
def test_very_long_sums_of_16_bit_results(side):
    """Positive terms, 2^23 of them in fp16, where half a step of the result is 2^-12 to 2^-11 of it.  A stretch of 1024 terms goes through 64 + 20
    additions of the tensor core, each off by at most a whole step of fp32, 2 U; the sums of stretches are added in fp32, each addition off by U, 512 of
    them in a line in each of the 16 parts of so long a sum, and then the parts: at most (168 + 512 + 16) U = 4.2e-5 of the result."""
    g = torch.Generator(device="cuda").manual_seed(15)
    some = lambda *s: (0.5 + 0.5 * torch.rand(*s, device="cuda", generator=g)).to(F16)  # noqa: E731
    long = 1 << 23
    if side == "rows":
        x, w, dy = some(long, 8), some(16, 8).requires_grad_(), some(long, 16) * 2.0 ** -8
        got = torch.autograd.grad(ops.linear(x, w), w, dy)[0]
        want = dy.double().t() @ x.double()
    else:
        x, w = some(20, long), some(8, long) * 2.0 ** -8
        got = ops.linear(x, w)
        want = x.double() @ w.double().t()
    assert want.min() > 1000 and want.max() < 60000
    assert ((got.double() - want).abs() <= (half_step(F16) + 4.2e-5) * want).all()
    # What is lost to an accumulator that is cut off lies on one side; a rounding to nearest is 0.29 of a step off, on either side: five of its standard deviations.
    step = torch.finfo(F16).eps * 2.0 ** torch.floor(torch.log2(want))
    assert abs(float(((got.double() - want) / step).mean())) <= 0.29 * 5 / want.numel() ** 0.5 + 4.2e-5 * 2 / torch.finfo(F16).eps


@pytest.mark.gpu
@pytest.mark.parametrize("kind,k", [(F16, 8200), (F16, 20001), (BF16, 65608)])
@pytest.mark.parametrize("act,residual", [(None, None), ("gelu_tanh", None), ("silu", "same")])
def test_long_sums_of_many_tiles_in_16_bits(kind, k, act, residual):
    """Sums in stretches with everything that follows a product, the argument that is kept among it, and rows that TMA does not store.  Enough tiles that
    no sum is shared out."""
    for m, n in ((2300, 2040), (2190, 2043)):
        assert _lib.cuda().hc_linear_bytes(m, k, n) == 0
        x, w, b, r, dy = make(m, k, n, kind, 16, kind, kind if residual else None)
        check(x, w, b, r, dy, act)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(5, 96, 50), (300, 264, 200), (77, 65, 129), (40, 200, 6144), (2500, 64, 96)])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
@pytest.mark.parametrize("dy_size,operand_size", [(2.0 ** -30, 2.0 ** 10), (2.0 ** 24, 2.0 ** -12), (2.0 ** 100, 2.0 ** -14), (2.0 ** -126, 1.0), (1.0, 1.0), (0.0, 1.0)])
def test_fp32_gradients_beyond_fp16(m, k, n, act, dy_size, operand_size):
    """An fp32 gradient enters fp16 products times a power of two, which takes its largest value to 2^13 at least: what is rounded there is 2^-11 of a value,
    or 2^-25 2^-13 of the largest one.  Only what fp16 does not hold of the result itself is infinite or 0."""
    g = torch.Generator().manual_seed(m)
    x, w, b = (torch.randn(*s, generator=g).to(F16).cuda() for s in ((m, k), (n, k), (n,)))
    dy = (torch.randn(m, n, generator=g) * dy_size).cuda()
    grown = [(x * operand_size).to(F16).requires_grad_(), (w * operand_size).to(F16).requires_grad_(), b.requires_grad_()]
    y = ops.linear(*grown, activation=act, out_dtype=F32)
    got = torch.autograd.grad(y, grown, dy)
    X, W, B = (v.detach().double() for v in grown)
    z = X @ W.t() + B
    ez = sums(k) * (X.abs() @ W.abs().t()) + U * z.abs()
    D = dy.double()
    if act is None:
        dz, e = D, torch.zeros_like(D)
    else:
        z = z.requires_grad_()
        (slope,) = torch.autograd.grad(ACT[act](z).sum(), (z,))
        z = z.detach()
        dz, e = D * slope, D.abs() * (0.8 * (half_step(F16) * z.abs() + ez + least(F16)) + 8 * U)
    e = e + half_step(F16) * dz.abs() + 2.0 ** -38 * D.abs().max()
    for have, left, right, el in ((got[0], dz, W, e), (got[1], dz.t(), X, e.t())):
        want = left @ right
        room = 1.01 * (el @ right.abs() + sums(left.shape[1]) * ((left.abs() + el) @ right.abs()) + half_step(F16) * want.abs()) + least(F16)
        clear = want.abs() + room < 65500
        assert torch.isfinite(have[clear]).all() and ((have.double() - want).abs() <= room)[clear].all()
        assert torch.isinf(have[want.abs() - room > 65540]).all()
        if dy_size == 0.0:
            assert not have.any()
    want = dz.sum(0)
    room = 1.01 * (e.sum(0) + (m + 64) * U * (dz.abs() + e).sum(0) + half_step(F16) * want.abs()) + least(F16)
    clear = want.abs() + room < 65500
    assert ((got[2].double() - want).abs() <= room)[clear].all()


@pytest.mark.gpu
def test_fp32_gradients_beyond_fp16_that_are_not_finite():
    """What is infinite or not a number in one row, and one column, has no part in the power that the others are taken times."""
    g = torch.Generator().manual_seed(3)
    x, w = torch.randn(200, 64, generator=g).to(F16).cuda().requires_grad_(), (torch.randn(96, 64, generator=g) * 2.0 ** 8).to(F16).cuda().requires_grad_()
    dy = (torch.randn(200, 96, generator=g) * 2.0 ** -28).cuda()
    dy[7, 9] = 0.0
    clean = torch.autograd.grad(ops.linear(x, w, out_dtype=F32), (x, w), dy)
    assert clean[0].any(1).all()
    for bad in (float("inf"), float("nan")):
        dy[7, 9] = bad
        dx, dw = torch.autograd.grad(ops.linear(x, w, out_dtype=F32), (x, w), dy)
        rows, columns = [i for i in range(200) if i != 7], [i for i in range(96) if i != 9]
        assert torch.equal(dx[rows], clean[0][rows]) and torch.equal(dw[columns], clean[1][columns])
        assert not torch.isfinite(dx[7]).all() and not torch.isfinite(dw[9]).all()


@pytest.mark.gpu
def test_fp32_gradients_of_any_size_in_a_graph():
    """The power of two is found anew in every replay."""
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(200, 64, generator=g).to(F16).cuda(), torch.randn(96, 64, generator=g).to(F16).cuda()
    dy = torch.randn(200, 96, generator=g).cuda()
    wide = torch.randn(200, 130, generator=g).cuda()[:, 3:99]  # rows with gaps

    def step():
        leaves = [v.detach().requires_grad_() for v in (x, w)]
        y = ops.linear(*leaves, out_dtype=F32)
        return (*torch.autograd.grad(y, leaves, dy, retain_graph=True), *torch.autograd.grad(y, leaves, wide))

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = step()
    for size in (2.0 ** 20, 2.0 ** -40, 2.0 ** 10):
        dy.mul_(size)
        wide.mul_(size)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(p, q) for p, q in zip(caught, want)) and want[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(5, 64, 40), (300, 264, 200)])
@pytest.mark.parametrize("out_dtype", [None, F32])
def test_infinite_gradients_of_what_relu_leaves_out(m, k, n, out_dtype):
    """Where its argument is not above 0 nothing depends on the result, whatever the gradient is there."""
    x, w, b, _, _ = make(m, k, n, BF16, 17)
    dy = torch.randn(m, n, generator=torch.Generator().manual_seed(18)).to(out_dtype or BF16).cuda()
    leaves = [v.detach().requires_grad_() for v in (x, w, b)]
    y = ops.linear(*leaves, activation="relu", out_dtype=out_dtype)
    off = y.detach() == 0
    assert off.any() and not off.all()
    want = torch.autograd.grad(y, leaves, torch.where(off, 0.0, dy), retain_graph=True)
    for bad in (float("inf"), -float("inf"), float("nan")):
        got = torch.autograd.grad(y, leaves, torch.where(off, bad, dy), retain_graph=True)
        assert all(torch.isfinite(p).all() and torch.equal(p, q) for p, q in zip(want, got))
