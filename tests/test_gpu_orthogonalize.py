"""The Newton-Schulz iteration against the same steps in 64 bits.

Tolerance, in units of the result's norm.  With r = 2^-11 / sqrt(3), the root mean square of an fp16 rounding: where singular
values are near 1 the polynomial of S is about -2.7, so a step's roundings of X, of the polynomial and of S come to 2.7 r, 2.7 r
and 2.2 r, 4.4 r together; the step before adds as much times the iteration's slope of at most 1.5, and so on: less than 12 r, 3.4e-3.
Rounding the result to bf16 adds at most 2^-8 / sqrt(3) = 2.3e-3.  Together 5.7e-3."""
import ctypes as C

import pytest
import torch

from tirocinio_triennale_b200 import _lib, ops

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
ROOM = 5.7e-3


def reference(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = g.double()
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    for _ in range(steps):
        s = x @ x.mT if x.shape[-2] <= x.shape[-1] else x.mT @ x
        q = b * s + c * s @ s
        x = a * x + (q @ x if x.shape[-2] <= x.shape[-1] else x @ q)
    return x


def check(g, room=ROOM, **kw):
    got, want = ops.orthogonalize(g, **kw), reference(g, **kw)
    assert got.dtype == torch.bfloat16 and got.shape == g.shape and not got.requires_grad
    d = got.double() - want
    assert (torch.linalg.matrix_norm(d) <= room * torch.linalg.matrix_norm(want) + 1e-30).all()
    rms = want.square().mean((-2, -1), keepdim=True).sqrt()
    assert (d.abs() <= 8 * room * torch.maximum(rms, want.abs())).all()
    return got


def gaussian(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("height,width", [(1, 1), (1, 64), (64, 1), (8, 8), (32, 48), (64, 192), (192, 64), (100, 100), (128, 128), (129, 130), (131, 129), (127, 600), (500, 75), (255, 257), (16, 1000), (700, 33), (96, 340), (60, 2000), (768, 768), (300, 1100), (1030, 260)])
def test_sizes(height, width):
    # a few rows or columns: the matrix is next to orthogonal already, few roundings average out
    check(gaussian(height, width, seed=height), ROOM if min(height, width) > 1 else 8e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 192, 64), (3, 2, 70, 90), (5, 33, 200), (17, 64, 64), (1, 300, 200)])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16, torch.float16])
def test_batches_and_types(shape, kind):
    g = gaussian(*shape, seed=1).to(kind)
    got = check(g)
    flat, each = g.reshape(-1, *shape[-2:]), got.reshape(-1, *shape[-2:])
    for i in range(flat.shape[0]):
        assert torch.equal(ops.orthogonalize(flat[i]), each[i])


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [1, 4, 40])
@pytest.mark.parametrize("height,width", [(300, 200), (200, 640)])
def test_few_directions(rank, height, width):
    """What is rounded off must not come up in the directions that the matrix does not have."""
    falling = 1 / torch.arange(1, rank + 1, device="cuda")
    check((gaussian(height, rank, seed=2) * falling) @ gaussian(rank, width, seed=3))


@pytest.mark.gpu
def test_scale_does_not_count_and_extremes():
    g = gaussian(90, 140, seed=4)
    want = ops.orthogonalize(g)
    for k in (-60, 40, 100):
        # eps is 1e-7 of a norm of 112, or of 112 times 2^-60: it goes by the reference
        check(g * 2.0 ** k)
    assert torch.equal(ops.orthogonalize(g * 2.0 ** 40, eps=0.0), ops.orthogonalize(g, eps=0.0))
    zero = ops.orthogonalize(torch.zeros(3, 40, 50, device="cuda"))
    assert not zero.any()
    mixed = torch.stack([g, torch.full_like(g, float("nan")), torch.zeros_like(g), g])
    got = ops.orthogonalize(mixed)
    assert torch.equal(got[0], want) and torch.equal(got[3], want) and torch.isnan(got[1]).all() and not got[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("height,width", [(200, 300), (300, 200), (70, 45)])
def test_terms_one_by_one(height, width):
    g = gaussian(height, width, seed=5)
    x = g.double() / torch.linalg.matrix_norm(g.double())
    got = ops.orthogonalize(g, steps=1, coefficients=(1.0, 0.0, 0.0), eps=0.0).double()
    # X from two fp16 numbers: 2^-22 of an entry, and 2^-36 where hi is below fp16's normal numbers; then one rounding to bf16
    assert ((got - x).abs() <= (2.0 ** -8 + 2.0 ** -20) * x.abs() + 2.0 ** -34).all()
    for k in (1, 2):
        c = (0.0, 1.0, 0.0) if k == 1 else (0.0, 0.0, 1.0)
        got = ops.orthogonalize(g, steps=1, coefficients=c, eps=0.0).double()
        want = reference(g, 1, c, 0.0)
        # entries of the sums are rounded to fp16: 2^-11 and, below its normal numbers, 2^-25 each
        s = x @ x.mT if height <= width else x.mT @ x
        if k == 2:
            s = s @ s
        off = (2.0 ** -10 * s.abs() + (2.0 ** -25 + 2.0 ** -10 * s.abs().max()))
        room = off @ x.abs() if height <= width else x.abs() @ off
        assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 2 * room).all()


@pytest.mark.gpu
def test_steps_and_coefficients():
    g = gaussian(60, 100, seed=6)
    check(g, steps=3)
    check(g, 8e-3, steps=8, coefficients=(1.875, -1.25, 0.375))
    s = torch.linalg.svdvals(ops.orthogonalize(g, steps=12, coefficients=(1.875, -1.25, 0.375)).double())
    assert ((s - 1).abs() < 0.02).all()


@pytest.mark.gpu
def test_views():
    wide = gaussian(4, 90, 160, seed=7)
    for g in (wide[:, 3:73, 5:128], wide.mT, wide[::2, :, :80], wide[..., ::2], wide.transpose(0, 1), wide[:1].expand(3, 90, 160)):
        assert torch.equal(ops.orthogonalize(g), ops.orthogonalize(g.contiguous()))
    assert ops.orthogonalize(torch.empty(0, 5, 6, device="cuda")).shape == (0, 5, 6)


@pytest.mark.gpu
def test_same_bits_every_time_other_streams_and_graphs():
    g = gaussian(3, 200, 456, seed=8)
    want = ops.orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = ops.orthogonalize(g)
    again = ops.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.orthogonalize(g)))
    g.copy_(g.flip(0))
    other = ops.orthogonalize(g)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, there) and torch.equal(want, again)
    assert all(torch.equal(other, caught) for _, caught in graphs)
    assert ops.train_status() == 0


@pytest.mark.gpu
def test_refusals():
    g = torch.zeros(8, 8, device="cuda")
    for bad in (lambda: ops.orthogonalize(g.double()), lambda: ops.orthogonalize(g[0]), lambda: ops.orthogonalize(g[:, :0]), lambda: ops.orthogonalize(g, steps=0),
                lambda: ops.orthogonalize(g, steps=101), lambda: ops.orthogonalize(g, eps=-1.0), lambda: ops.orthogonalize(g, coefficients=(1, 2)), lambda: ops.orthogonalize(g.cpu())):
        with pytest.raises(ValueError):
            bad()


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        ops.orthogonalize(torch.ones(4, 4))
    lib = _lib.cuda()
    p = C.c_void_p(4096)  # never read: every call below is refused before anything is launched
    good = dict(g=p, type=0, batch=2, h=16, w=24, s=24, bs=384, out=p, steps=5, a=3.0, b=-4.0, c=2.0, eps=1e-7, scratch=p, bytes=1 << 30)

    def call(**kw):
        return lib.hc_orthogonalize(*{**good, **kw}.values(), None)

    for kw in (dict(type=3), dict(batch=65536), dict(h=0), dict(w=0), dict(w=1 << 24, s=1 << 24), dict(s=23), dict(steps=0), dict(steps=101), dict(eps=-1.0), dict(g=None), dict(out=None),
               dict(scratch=None), dict(scratch=C.c_void_p(4100)), dict(bytes=100)):
        assert call(**kw) == 4, kw
    assert call(batch=0) == 0 and lib.hc_orthogonalize_bytes(0, 4, 4) == 0
    assert lib.hc_orthogonalize_bytes(12, 2304, 768) >= 12 * (3 * 2304 * 768 + 2 * 768 * 768) * 2


GROWING = [((3.0, 0.0, 0.0), 12), ((2.0, 1.0, 0.0), 4), ((-3.0, 0.0, 0.0), 12), ((1.0, 0.0, 300.0), 2), ((1.0, 70000.0, 0.0), 1), ((float("nan"), 0.0, 0.0), 2), ((1.0, float("inf"), 0.0), 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 60), (200, 300), (300, 200)])
def test_iterations_that_leave_the_range_of_their_operands(shape):
    """X, S and the polynomial are held in fp16: coefficients that may carry them beyond it are refused, those that do not give what the formula gives."""
    g = gaussian(*shape, seed=9)
    for coefficients, steps in GROWING:
        with pytest.raises(ValueError, match="float16"):
            ops.orthogonalize(g, steps=steps, coefficients=coefficients)
    for coefficients, steps in (((3.0, 0.0, 0.0), 5), ((-3.0, 0.0, 0.0), 4), ((1.0, 60000.0, 0.0), 1), ((2.0, 1.0, 0.0), 3)):
        got, want = ops.orthogonalize(g, steps=steps, coefficients=coefficients).double(), reference(g, steps, coefficients)
        # A step's result has, in units of r above, the rounding of X as an operand of either product with S (2), of S and of the polynomial: 4 r in the terms
        # with S, and moves with X by the polynomial's slope over its value, 3 at most where there is no S S term: (4 + 3 (4 + 3 4)) r = 52 r over three steps, and bf16.
        assert torch.linalg.matrix_norm(got - want) <= (52 * 2.0 ** -11 / 3 ** 0.5 + 2.3e-3) * torch.linalg.matrix_norm(want)


def test_coefficients_refused_without_a_gpu():
    lib = _lib.cuda()
    p = C.c_void_p(4096)  # never read: every call below is refused before anything is launched
    for (a, b, c), steps in GROWING:
        for h, w in ((16, 24), (400, 300)):
            assert lib.hc_orthogonalize(p, 0, 2, h, w, w, h * w, p, steps, a, b, c, 1e-7, p, 1 << 30, None) == 4, (a, b, c, steps)


def test_sizes_whose_memory_no_number_holds():
    """Scratch memory of more bytes than 64 bits count is refused, not counted anew from 0."""
    lib = _lib.cuda()
    p = C.c_void_p(4096)
    for batch, h, w in ((65535, 1 << 23, 1 << 23), (65535, (1 << 24) - 1, (1 << 24) - 1), (65535, 5305712, 5305712)):
        assert lib.hc_orthogonalize_bytes(batch, h, w) == 0
        assert lib.hc_orthogonalize(p, 0, batch, h, w, w, 0, p, 5, 3.0, -4.0, 2.0, 1e-7, p, (1 << 64) - 1, None) == 4
    # a matrix that a GPU holds is still counted
    assert lib.hc_orthogonalize_bytes(1, 1 << 16, 1 << 16) >= 5 * (1 << 33)


@pytest.mark.gpu
@pytest.mark.parametrize("height,width", [(32, 1 << 22), (1 << 20, 64), (700, 70001), (20000, 260)])
def test_long_sides(height, width):
    """S is a sum over the long side, of positive terms in its diagonal; its precision does not go with the length."""
    check(torch.randn(height, width, device="cuda", generator=torch.Generator(device="cuda").manual_seed(10)))
