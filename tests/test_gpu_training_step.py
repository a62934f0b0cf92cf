"""A step of the model through attention, the loss without logits and AdamW in one launch, all of them together: in a graph, in the trainer, resumed."""
import argparse
import copy

import pytest
import torch

from mp_util import run_ranks
from tirocinio_triennale_b200 import ops
from tirocinio_triennale_b200.models import GPT2, AdamW, GPT2Config


def _model(**kw):
    cfg = GPT2Config.tiny()
    cfg.fused, cfg.logits, cfg.attention, cfg.window, cfg.sinks = True, False, "own", 12, 2
    for k, v in kw.items():
        setattr(cfg, k, v)
    torch.manual_seed(0)
    return GPT2(cfg).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_step_in_a_graph(bits):
    """Whole steps captured and replayed: the same weights as after the same steps outside.  Torch's embeddings add their gradients in any order, which moves everything behind
    the first step a little.  (With a graph of the same parameters alive that was made outside, torch itself refuses the capture: their accumulation belongs to that graph's stream.)"""
    tok = torch.randint(0, 257, (2, 33), generator=torch.Generator().manual_seed(2)).cuda()
    inputs = [tok.clone(), tok.flip(0).clone(), (tok + 3) % 257]

    def steps(model, opt):
        held = tok.clone()

        def step():
            loss = model(held[:, :-1], held[:, 1:])
            opt.zero_grad(set_to_none=True)
            loss.backward()
            opt.step()

        return held, step

    eager = _model()
    opt = AdamW(eager.parameters(), lr=1e-2, bits=bits, capturable=True)
    held, step = steps(eager, opt)
    for t in [inputs[0]] * 3 + inputs:
        held.copy_(t)
        step()
    caught = _model()
    opt = AdamW(caught.parameters(), lr=1e-2, bits=bits, capturable=True)
    held, step = steps(caught, opt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    held.copy_(inputs[0])
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in inputs:
        held.copy_(t)
        graph.replay()
    torch.cuda.synchronize()
    for (name, a), b in zip(eager.named_parameters(), caught.parameters()):
        assert (a - b).norm() <= 1e-2 * a.norm() + 1e-3, name
    assert ops.train_status() == 0


@pytest.mark.gpu
def test_gradients_of_the_whole_model():
    """All parameters' gradients against the plain model's in 64 bits: 40 roundings of at most 2^-8, in relative 2-norm."""
    import torch.nn.functional as F

    model = _model(n_layer=2, d_model=128, n_head=2, vocab_size=1003, seq_len=200)
    cfg = copy.copy(model.cfg)
    cfg.fused, cfg.attention, cfg.logits = False, "torch", True
    plain = GPT2(cfg).cuda()
    plain.load_state_dict(model.state_dict())
    plain = plain.double()
    tok = torch.randint(0, 1003, (2, 201), generator=torch.Generator().manual_seed(3)).cuda()
    loss = model(tok[:, :-1], tok[:, 1:])
    loss.backward()
    want = F.cross_entropy(plain(tok[:, :-1]).reshape(-1, 1003), tok[:, 1:].reshape(-1))
    want.backward()
    room = 40 * 2.0 ** -8
    assert abs(loss.item() - want.item()) <= room * want.item()
    for (name, p), q in zip(model.named_parameters(), plain.named_parameters()):
        q = q[1]
        scale = q.grad.norm() if not name.endswith("qkv.bias") else model.blocks[0].qkv.weight.grad.double().norm()
        assert (p.grad.double() - q.grad).norm() <= room * scale, name
    assert ops.train_status() == 0


def test_options_that_do_not_go_together():
    cfg = GPT2Config.tiny()
    cfg.attention = "own"
    with pytest.raises(ValueError, match="attention"):
        GPT2(cfg)
    cfg.attention = "other"
    with pytest.raises(ValueError, match="attention"):
        GPT2(cfg)


def test_window_without_a_gpu():
    """The plain model's window is the mask that the operator's documentation gives."""
    cfg = GPT2Config.tiny()
    cfg.window, cfg.sinks = 5, 2
    torch.manual_seed(0)
    model = GPT2(cfg)
    q, k, v = (torch.randn(1, 2, 20, 32, generator=torch.Generator().manual_seed(i)) for i in range(3))
    p = torch.arange(20)[:, None]
    j = torch.arange(20)[None]
    s = (q @ k.mT / 32 ** 0.5).masked_fill(~((j <= p) & ((p - j < 5) | (j < 2))), -float("inf"))
    assert (model.blocks[0].attend(q, k, v) - torch.softmax(s, -1) @ v).abs().max() < 1e-5


def _trainer(rank, world, prefix):
    from tirocinio_triennale_b200.models import train_dp

    args = argparse.Namespace(model="tiny", steps=3, warmup=1, batch=2, seq=32, eb=1e-6, lr=1e-3, bucket_mb=0.05, cpu=False, save=prefix, resume=None, save_compressed_eb=0.0, fused=True,
                              optimizer="adamw", muon_lr=0.02, adam_bits=8, attention="own", window=9, sinks=1, no_logits=True)
    for compressed in (True, False):
        out = train_dp.run(args, compressed, rank, world, torch.device("cuda", 0))
        assert out["steps_done"] == 4 and out["last_loss_rank0"] == out["last_loss_rank0"]
    args.resume, args.save, args.optimizer = prefix, None, "adamw"
    out = train_dp.run(args, True, rank, world, torch.device("cuda", 0))
    assert out["steps_done"] == 8
    assert ops.train_status() == 0


@pytest.mark.gpu
def test_trainer_with_all_of_them(tmp_path):
    run_ranks(_trainer, 1, backend="nccl", args=(str(tmp_path / "ck"),))
