"""The operators of the training step together: the model that runs through them, its gradients, the Muon update, the trainer."""
import argparse
import copy
import ctypes as C

import pytest
import torch
import torch.nn.functional as F

from mp_util import run_ranks
from tirocinio_triennale_b200 import _lib, ops
from tirocinio_triennale_b200.models import GPT2, GPT2Config, Muon, muon_with_adamw
from tirocinio_triennale_b200.models.muon import Optimizers


def _pair(**kw):
    cfg = GPT2Config.tiny()
    for k, v in kw.items():
        setattr(cfg, k, v)
    torch.manual_seed(0)
    plain = GPT2(cfg).cuda()
    cfg = copy.copy(cfg)
    cfg.fused = True
    fused = GPT2(cfg).cuda()
    fused.load_state_dict(plain.state_dict())
    return plain.double(), fused


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [dict(), dict(d_model=96, n_head=3, vocab_size=1001, n_layer=1), dict(d_model=128, n_head=4, vocab_size=50257)])
def test_model_through_the_operators(shape):
    """Each of the two layers rounds some 8 tensors to bf16 on the way forward and as many on the way back, the head 4 and 4: 40
    roundings of at most 2^-8 each, in relative 2-norm."""
    plain, fused = _pair(**shape)
    room = 40 * 2.0 ** -8
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, plain.cfg.vocab_size, (3, 33), generator=g).cuda()
    idx, targets = tok[:, :-1], tok[:, 1:].clone()
    targets[0, :5] = -100
    logits = fused(idx)
    want = plain(idx)
    assert logits.dtype == torch.bfloat16 and (logits.double() - want).norm() <= room * want.norm()
    loss = fused(idx, targets)
    loss.backward()
    exact = F.cross_entropy(want.reshape(-1, want.shape[-1]), targets.reshape(-1))
    exact.backward()
    assert abs(loss.item() - exact.item()) <= room * exact.item()
    for (name, p), q in zip(fused.named_parameters(), plain.parameters()):
        assert p.grad.dtype == p.dtype == torch.float32 and p.grad.shape == p.shape
        # a key's bias moves all scores of a query alike: its gradient is 0, and what stands there is rounding alone
        scale = q.grad.norm() if not name.endswith("qkv.bias") else fused.blocks[0].qkv.weight.grad.double().norm()
        assert (p.grad.double() - q.grad).norm() <= room * scale, name
    assert ops.train_status() == 0


@pytest.mark.gpu
def test_model_in_a_graph():
    """A step's forward and backward pass captured and replayed on other tokens gives what it gives outside."""
    _, model = _pair()
    tok = torch.randint(0, 257, (2, 33), generator=torch.Generator().manual_seed(2)).cuda()

    def step():
        model.zero_grad(set_to_none=True)
        loss = model(tok[:, :-1], tok[:, 1:])
        loss.backward()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    model.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = step()
    tok.copy_(tok.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    grads = [p.grad.clone() for p in model.parameters()]
    caught = caught.clone()
    for p in model.parameters():
        p.grad = None
    assert torch.equal(step(), caught)
    assert all((a - p.grad).norm() <= 1e-2 * a.norm() for a, p in zip(grads, model.parameters()))  # torch's attention may add in any order


def _reference_step(p, g, m, lr, momentum, decay, nesterov):
    m = momentum * m + g
    u = g + momentum * m if nesterov else m
    a, b, c = 3.4445, -4.7750, 2.0315
    x = u / (u.norm() + 1e-7)
    for _ in range(5):
        s = x @ x.T
        x = a * x + (b * s + c * s @ s) @ x
    return p * (1 - lr * decay) - lr * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * x, m


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_against_the_formulas(nesterov):
    g = torch.Generator().manual_seed(3)
    shapes = [(48, 96), (96, 48), (48, 96), (200, 130), (33, 7)]
    params = [torch.nn.Parameter(torch.randn(*s, generator=g).cuda()) for s in shapes]
    want = [(p.detach().double(), torch.zeros_like(p).double()) for p in params]
    opt = Muon(params, lr=0.05, momentum=0.9, weight_decay=0.1, nesterov=nesterov)
    for _ in range(3):
        for i, p in enumerate(params):
            p.grad = torch.randn(*shapes[i], generator=g).cuda()
            want[i] = _reference_step(want[i][0], p.grad.double(), want[i][1], 0.05, 0.9, 0.1, nesterov)
        opt.step()
    for p, (w, m) in zip(params, want):
        assert (opt.state[p]["momentum"].double() - m).norm() <= 1e-6 * m.norm()
        # three updates, each within 5.7e-3 of its norm (that of the iteration's test) and of norm lr sqrt(rank) sqrt(height / width)
        size = 3 * 0.05 * min(p.shape) ** 0.5 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * 1.2
        assert (p.detach().double() - w).norm() <= 8e-3 * size


@pytest.mark.gpu
def test_muon_with_adamw_state_and_refusals():
    _, model = _pair()
    opt = muon_with_adamw(model)
    muon, adam = opt.optimizers
    assert len(muon.param_groups[0]["params"]) == 8 and all(p.dim() == 2 for p in muon.param_groups[0]["params"])
    held = {id(p) for o in (muon, adam) for gr in o.param_groups for p in gr["params"]}
    assert held == {id(p) for p in model.parameters()} and id(model.wte.weight) in {id(p) for p in adam.param_groups[0]["params"]}
    tok = torch.randint(0, 257, (2, 33), generator=torch.Generator().manual_seed(4)).cuda()
    for _ in range(2):
        opt.zero_grad()
        model(tok[:, :-1], tok[:, 1:]).backward()
        opt.step()
    assert all(torch.isfinite(p).all() for p in model.parameters())
    again = muon_with_adamw(model)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    p = muon.param_groups[0]["params"][0]
    assert torch.equal(again.optimizers[0].state[p]["momentum"], muon.state[p]["momentum"])
    with pytest.raises(ValueError):
        again.load_state_dict(opt.state_dict()[:1])
    opt.zero_grad()
    opt.step()  # without gradients nothing moves


@pytest.mark.gpu
def test_gradients_have_no_gradients():
    x = torch.randn(20, 64, device="cuda", requires_grad=True)
    t = torch.zeros(20, dtype=torch.int64, device="cuda")
    h = x.detach().bfloat16().requires_grad_()
    for y, leaf in ((ops.layer_norm(x), x), (ops.linear(h, h), h), (ops.token_logprobs(x, t).logprobs, x)):
        (d,) = torch.autograd.grad(y.float().square().sum(), (leaf,), create_graph=True)
        with pytest.raises(RuntimeError, match="no gradients of their own"):
            d.sum().backward()
        assert torch.isfinite(d).all()


def test_refusals_without_a_gpu():
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(3, 3))], momentum=1.0)
    cfg = GPT2Config.tiny()
    cfg.fused = True
    with pytest.raises(ValueError, match="CUDA"):
        GPT2(cfg)(torch.zeros(1, 4, dtype=torch.int64))
    p = torch.nn.Parameter(torch.zeros(3, 3))
    p.grad = torch.zeros(3, 3)
    with pytest.raises(ValueError, match="CUDA"):
        Optimizers(Muon([p])).step()


def test_pointers_between_elements_are_refused():
    """Whatever a call reads or writes begins where its elements may; nothing below is launched."""
    lib = _lib.cuda()
    p, odd, half = (C.c_void_p(v) for v in (4096, 4097, 4098))
    big = 1 << 30

    def refused(name, good, **bad):
        fn = getattr(lib, name)
        for key, value in bad.items():
            assert fn(*{**good, key: value}.values(), None) == 4, (name, key)

    refused("hc_layer_norm", dict(x=p, xt=1, w=p, b=p, pt=0, y=p, yt=1, st=p, rows=4, width=16, eps=1e-5), w=half, b=half, st=half)
    refused("hc_layer_norm_backward", dict(dy=p, yt=1, x=p, xt=1, w=p, pt=0, st=p, dx=p, dw=p, db=p, rows=4, width=16, scratch=p, bytes=big), w=half, st=half, dx=half, dw=half,
            db=half, scratch=half)
    refused("hc_linear", dict(x=p, xs=16, w=p, ws=16, type=1, b=p, bt=0, r=p, rs=24, out=p, ot=0, os=24, z=p, zs=24, act=1, m=3, k=16, n=24, scratch=None, bytes=0), x=odd, w=odd,
            b=half, r=half, out=half, z=odd)
    refused("hc_linear_backward", dict(dy=p, dt=0, ds=24, z=p, zs=24, act=1, keep=1, x=p, xs=16, w=p, ws=16, type=1, dx=p, dxs=16, dw=p, dws=16, db=p, bt=0, m=32, k=16, n=24,
                                       scratch=p, bytes=big), dy=half, z=odd, dx=odd, dw=odd, db=half)
    refused("hc_token_logprobs", dict(x=p, type=1, rows=4, vocab=16, stride=16, tokens=p, ignore=-100, top=2, lp=p, h=p, tt=p, tl=p, st=p), x=odd, tokens=half, lp=half, h=half, tt=half,
            tl=half, st=half)
    refused("hc_token_logprobs_backward", dict(x=p, type=1, rows=4, vocab=16, stride=16, tokens=p, ignore=-100, st=p, a=p, b=p, d=p, ds=16), x=odd, tokens=half, st=half, a=half, b=half,
            d=odd)
    refused("hc_orthogonalize", dict(g=p, type=0, batch=2, h=16, w=24, s=24, bs=384, out=p, steps=5, a=3.0, b=-4.0, c=2.0, eps=1e-7, scratch=p, bytes=big), g=half, out=odd)


def _trainer(rank, world):
    from tirocinio_triennale_b200.models import train_dp

    args = argparse.Namespace(model="tiny", steps=3, warmup=1, batch=2, seq=32, eb=1e-6, lr=1e-3, bucket_mb=0.05, cpu=False, save=None, resume=None,
                              save_compressed_eb=0.0, fused=True, optimizer="muon", muon_lr=0.02)
    for compressed in (True, False):
        out = train_dp.run(args, compressed, rank, world, torch.device("cuda", 0))
        assert out["steps_done"] == 4 and out["last_loss_rank0"] == out["last_loss_rank0"]
        assert not compressed or out["compressed_calls"] > 0
    assert ops.train_status() == 0


@pytest.mark.gpu
def test_trainer_with_the_operators_and_compressed_gradients():
    run_ranks(_trainer, 1, backend="nccl")


def _calls(device):
    """Every operator as a function of one of its tensors, with that tensor: name, function, tensor."""
    f, h = torch.float32, torch.bfloat16
    g = torch.Generator().manual_seed(5)
    some = lambda *s, t=f: torch.randn(*s, generator=g).to(t).to(device)  # noqa: E731
    x, w, b = some(6, 16), some(16), some(16)
    xh, wh, bh, r = some(20, 16, t=h), some(24, 16, t=h), some(24), some(20, 24)
    logits, tokens = some(5, 33), torch.arange(5, device=device)
    return [("norm x", lambda v: ops.layer_norm(v, w, b), x), ("norm weight", lambda v: ops.layer_norm(x, v, b), w), ("norm bias", lambda v: ops.layer_norm(x, w, v), b),
            ("linear x", lambda v: ops.linear(v, wh, bh, residual=r), xh), ("linear weight", lambda v: ops.linear(xh, v, bh, residual=r), wh),
            ("linear bias", lambda v: ops.linear(xh, wh, v, residual=r), bh), ("linear residual", lambda v: ops.linear(xh, wh, bh, residual=v), r),
            ("logits", lambda v: ops.token_logprobs(v, tokens).logprobs, logits), ("update", lambda v: ops.orthogonalize(v), some(8, 12))]


def _refuses_what_it_cannot_do(device):
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    for name, call, v in _calls(device):
        with forward_ad.dual_level():
            for leaf in (v.clone(), v.clone().requires_grad_()):
                with pytest.raises(NotImplementedError, match="forward"):
                    call(forward_ad.make_dual(leaf, torch.ones_like(v)))
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(call, (v,), check_trace=False)
        for kind in ("real", "fake"):
            with pytest.raises(NotImplementedError):
                make_fx(call, tracing_mode=kind)(v)
        for transformed in (lambda v=v: torch.vmap(call)(torch.stack([v, v])), lambda v=v: torch.func.jvp(call, (v,), (v,)), lambda v=v: torch.func.grad(lambda u: call(u).float().sum())(v)):
            with pytest.raises(NotImplementedError):
                transformed()


def test_forward_mode_tracing_and_transforms_are_refused():
    """A result made outside of torch's dispatcher has no tangent, and a recording of the call would hold an allocation that nothing fills."""
    _refuses_what_it_cannot_do("cpu")


@pytest.mark.gpu
def test_forward_mode_tracing_and_transforms_are_refused_on_a_gpu():
    _refuses_what_it_cannot_do("cuda")
    assert ops.train_status() == 0


@pytest.mark.gpu
def test_gradients_with_a_tangent_are_refused():
    """Forward mode over the backward pass: a Hessian-vector product, of which the gradient's tangent would be lost."""
    import torch.autograd.forward_ad as forward_ad

    for name, call, v in _calls("cuda"):
        if name in ("update", "linear residual"):  # no gradient; one that is handed through
            continue
        leaf = v.clone().requires_grad_()
        y = call(leaf)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward"):
                torch.autograd.grad(y, leaf, dual)


@pytest.mark.gpu
def test_views_that_are_the_negative_of_what_lies_there():
    """The imaginary part of a conjugate is such a view; so can gradients be."""
    for name, call, v in _calls("cuda"):
        want = call((-v).contiguous())
        assert torch.equal(call(torch._neg_view(v)), want), name
        if name == "update":
            continue
        leaf = v.clone().requires_grad_()
        y = call(leaf)
        dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(6)).to(y.dtype).cuda()
        (want,) = torch.autograd.grad(y, leaf, -dy, retain_graph=True)
        (got,) = torch.autograd.grad(y, leaf, torch._neg_view(dy))
        assert torch.equal(got, want), name
        leaf = torch._neg_view(v.clone()).requires_grad_()
        (got,) = torch.autograd.grad(call(leaf), leaf, dy)
        leaf = (-v).requires_grad_()
        assert torch.equal(got, torch.autograd.grad(call(leaf), leaf, dy)[0]), name


def _trainer_with_status(rank, world, status, prefix):
    import os

    from tirocinio_triennale_b200.models import train_dp

    asked = []

    def train_status(device=None, clear=True):
        asked.append(device)
        return status if rank == world - 1 else 0  # of one rank; all of them end

    train_dp.train_status = train_status
    model = train_dp.GPT2

    def plain(cfg):  # the operators need a GPU; what is tested is what the trainer makes of their status
        cfg = copy.copy(cfg)
        cfg.fused = False
        return model(cfg)

    train_dp.GPT2 = plain
    args = argparse.Namespace(model="tiny", steps=2, warmup=1, batch=2, seq=16, eb=1e-6, lr=1e-3, bucket_mb=0.05, cpu=True, save=prefix, resume=None, save_compressed_eb=0.0,
                              fused=True, optimizer="adamw", muon_lr=0.02)
    if status:
        with pytest.raises(RuntimeError, match="operators"):
            train_dp.run(args, True, rank, world, torch.device("cpu"))
    else:
        train_dp.run(args, True, rank, world, torch.device("cpu"))
    assert asked and os.path.exists("%s.compressed.rank%d" % (prefix, rank)) == (status == 0)


@pytest.mark.parametrize("world", [1, 2])
@pytest.mark.parametrize("status", [0, 3])
def test_a_wait_that_ran_out_ends_the_trainer_on_all_ranks(status, world, tmp_path):
    run_ranks(_trainer_with_status, world, backend="gloo", args=(status, str(tmp_path / "ck")))


def test_a_module_built_for_another_torch_is_built_anew(tmp_path, monkeypatch):
    """What the native front end was compiled against is in its name; another torch's classes lie differently."""
    from tirocinio_triennale_b200 import _build

    monkeypatch.setattr(_build, "LIBDIR", tmp_path)
    made = []

    def run(cmd):
        made.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return ""

    monkeypatch.setattr(_build, "_run", run)
    lib = _build.build_torch()
    assert lib.exists() and len(made) == 1
    assert _build.build_torch() == lib and len(made) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9+cu999")
    other = _build.build_torch()
    assert _build.build_torch() == other != lib and len(made) == 2
    monkeypatch.undo()
    monkeypatch.setattr(_build, "LIBDIR", tmp_path)
    monkeypatch.setattr(_build, "_run", run)
    assert _build.build_torch() == lib and len(made) == 2
    lib.unlink()
    assert _build.build_torch() == lib and len(made) == 3


def test_muon_with_adamw_where_one_of_them_has_nothing():
    """A model without linear layers, and one of nothing but their matrices."""
    one = muon_with_adamw(torch.nn.LayerNorm(8))
    assert [type(o) for o in one.optimizers] == [torch.optim.AdamW]
    other = muon_with_adamw(torch.nn.Linear(8, 8, bias=False), lr=0.5)
    assert [type(o) for o in other.optimizers] == [Muon] and other.optimizers[0].param_groups[0]["lr"] == 0.5
    other.load_state_dict(other.state_dict())
    with pytest.raises(ValueError):
        one.load_state_dict([])
