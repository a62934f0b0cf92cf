"""A process's first call, captured: what a launcher asks the runtime once does not disturb the capture.  And a step that raises has changed nothing."""
import subprocess
import sys

import pytest
import torch

from tirocinio_triennale_b200 import ops

FIRST = """
import torch
from tirocinio_triennale_b200 import ops
g = torch.Generator().manual_seed(0)
some = lambda *s: torch.randn(*s, generator=g).to(torch.%s).cuda()
q, k, v, dout = (some(2, 3, 200, %d) for _ in range(4))
x, w = some(100, 64), some(300, 64)
t = torch.randint(0, 300, (100,), generator=g).cuda()
leaves = [a.requires_grad_() for a in (q, k, v, x, w)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    o = ops.attention(q, k, v)
    loss = ops.linear_cross_entropy(x, w, t)
    got = torch.autograd.grad((o, loss), leaves, (dout, torch.ones_like(loss)))
graph.replay()
torch.cuda.synchronize()
want_o = ops.attention(q, k, v)
want_loss = ops.linear_cross_entropy(x, w, t)
want = torch.autograd.grad((want_o, want_loss), leaves, (dout, torch.ones_like(loss)))
assert torch.equal(o, want_o) and torch.equal(loss, want_loss) and all(torch.equal(a, b) for a, b in zip(got, want))
assert ops.train_status() == 0
print("done")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bfloat16", "float16"])
@pytest.mark.parametrize("d", [64, 128])
def test_first_calls_in_a_capture(kind, d):
    r = subprocess.run([sys.executable, "-c", FIRST % (kind, d)], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stdout + r.stderr


@pytest.mark.gpu
def test_a_step_that_raises_has_changed_nothing():
    """Tensors of inference mode may not be changed outside of it: said before the step is launched."""
    for inference in range(3):
        made = []
        for i in range(3):
            with torch.inference_mode(i == inference):
                made.append(torch.ones(1000, device="cuda"))
        grad = torch.ones(1000, device="cuda")
        p, m, v = made
        with pytest.raises(RuntimeError, match="[Ii]nference"):
            ops.adamw_step([p], [grad], [m], [v], step=1, lr=0.5)
        torch.cuda.synchronize()
        with torch.inference_mode():
            assert all((t == 1).all() for t in made)
