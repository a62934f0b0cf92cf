"""A captured step repeats what it did: state that began in it would begin again at each replay, and a step counted by the host would stay where it is.  Both are refused."""
import pytest
import torch

from tirocinio_triennale_b200.models import AdamW


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_that_cannot_be_replayed(bits):
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.full_like(p, 0.5)
    torch.cuda.synchronize()
    for capturable, match in ((False, "capturable"), (True, "before")):
        opt = AdamW([p], bits=bits, capturable=capturable)
        if not capturable:
            opt.step()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=match):
            with torch.cuda.graph(graph):
                opt.step()
        assert capturable is False or (not opt.state[p] and "steps" not in opt.param_groups[0])
        torch.cuda.synchronize()
    opt.step()  # outside it begins
    before = p.detach().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    assert torch.equal(p, before)
    graph.replay()
    torch.cuda.synchronize()
    assert int(opt.param_groups[0]["steps"]) == 2 and not torch.equal(p, before)


def test_refusals_without_a_gpu(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    p = torch.nn.Parameter(torch.ones(300))
    p.grad = torch.ones(300)
    for capturable, match in ((False, "capturable"), (True, "before")):
        opt = AdamW([p], capturable=capturable)
        with pytest.raises(RuntimeError, match=match):
            opt.step()
        assert not opt.state[p] and "steps" not in opt.param_groups[0]
