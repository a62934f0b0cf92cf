"""Calls from a thread that has called nothing of CUDA yet: the device's context is not current in it, and memory from the cache makes nothing of the runtime current either."""
import threading

import pytest
import torch

from tirocinio_triennale_b200 import ops


def _in_a_new_thread(call):
    got = []

    def run():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001
            got.append(e)

    for _ in range(2):  # the second finds its memory in the cache
        t = threading.Thread(target=run)
        t.start()
        t.join()
    for g in got:
        if isinstance(g, Exception):
            raise g
    return got[-1]


@pytest.mark.gpu
def test_products_in_a_new_thread():
    g = torch.Generator().manual_seed(0)
    x, w = (torch.randn(n, 64, generator=g).bfloat16().cuda() for n in (40, 48))
    want = ops.linear(x, w)
    assert torch.equal(_in_a_new_thread(lambda: ops.linear(x, w)), want)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    y = ops.linear(*leaves)
    want = torch.autograd.grad(y, leaves, y.detach(), retain_graph=True)
    got = _in_a_new_thread(lambda: torch.autograd.grad(y, leaves, y.detach(), retain_graph=True))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    u = torch.randn(40, 300, generator=g).cuda()
    assert torch.equal(_in_a_new_thread(lambda: ops.orthogonalize(u)), ops.orthogonalize(u))


@pytest.mark.gpu
def test_attention_loss_and_step_in_a_new_thread():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(1, 2, 130, 64, generator=g).bfloat16().cuda()
    assert torch.equal(_in_a_new_thread(lambda: ops.attention(q, q, q)), ops.attention(q, q, q))
    x, w = (torch.randn(n, 64, generator=g).bfloat16().cuda() for n in (40, 300))
    t = torch.arange(40, device="cuda")
    assert torch.equal(_in_a_new_thread(lambda: ops.linear_cross_entropy(x, w, t)), ops.linear_cross_entropy(x, w, t))
    p, d, m, v = (torch.ones(1000, device="cuda") for _ in range(4))
    _in_a_new_thread(lambda: ops.adamw_step([p], [d], [m], [v], step=1))
    a, b, c = (torch.ones(1000, device="cuda") for _ in range(3))
    for _ in range(2):
        ops.adamw_step([a], [d], [b], [c], step=1)
    assert torch.equal(a, p) and torch.equal(b, m) and torch.equal(c, v)
