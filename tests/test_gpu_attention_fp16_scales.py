"""Gradients of attention in fp16: a sequence's, and a key head's, are what they are whatever else is in the batch."""
import pytest
import torch

from tirocinio_triennale_b200 import ops

F16 = torch.float16


def gradients(q, k, v, dout, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(ops.attention(*leaves, **kw), leaves, dout)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 80, 128])
@pytest.mark.parametrize("heads,kv,queries,keys,window", [(4, 2, 200, 200, None), (6, 2, 65, 300, 100), (3, 3, 1, 77, None), (2, 1, 513, 513, None)])
def test_others_in_the_batch_change_nothing(heads, kv, queries, keys, window, d):
    """The same call but for the second sequence, or for the last key head, whose upstream gradients and values are 2^10 times as large: the same bits for the others."""
    g = torch.Generator().manual_seed(d + keys)
    some = lambda n, h: torch.randn(2, n, h, d, generator=g).to(F16).cuda().transpose(1, 2)
    q, k, v, dout = some(queries, heads), some(keys, kv), some(keys, kv), some(queries, heads) * 2.0 ** -8
    base = gradients(q, k, v, dout, window=window)
    group = heads // kv
    for what in ("sequence", "head"):
        if what == "head" and kv == 1:
            continue
        for grows in ("dout", "v", "both"):
            dout2, v2 = dout.clone(), v.clone()
            if what == "sequence":
                if grows != "v":
                    dout2[1] *= 2.0 ** 10
                if grows != "dout":
                    v2[1] *= 2.0 ** 10
            else:
                if grows != "v":
                    dout2[:, -group:] *= 2.0 ** 10
                if grows != "dout":
                    v2[:, -1] *= 2.0 ** 10
            for a, b in zip(base, gradients(q, k, v2, dout2, window=window)):
                n = a.shape[1] // kv
                assert torch.equal(*((t[0] for t in (a, b)) if what == "sequence" else (t[:, :-n] for t in (a, b)))), (what, grows)
    assert ops.train_status() == 0


@pytest.mark.gpu
def test_small_gradients_beside_large_ones():
    """Upstream gradients of two sequences 2^20 apart: the small one's dQ and dK are as near the formula's, relative to their size, as the large one's.
    Roundings to fp16: of P and dS, of O in delta, of the result, 2^-11 each of what the result's terms add up to (the norm of 1000 of them: far less than 8 of these of the whole), and dS below 2^-24
    of a power of two that is at least 2^-3 of the largest it can be, 2 max|dO| max|V|."""
    g = torch.Generator().manual_seed(3)
    some = lambda: torch.randn(2, 1000, 2, 64, generator=g).transpose(1, 2)
    q, k, v, dout = (t.to(F16).cuda() for t in (some(), some(), some(), some() * torch.tensor([2.0 ** -10, 2.0 ** 10])[:, None, None, None]))
    got = gradients(q, k, v, dout)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    s = (leaves[0] @ leaves[1].mT) / 8
    s = s.masked_fill(~torch.ones(1000, 1000, device="cuda").tril().bool(), -torch.inf)
    want = torch.autograd.grad(torch.softmax(s, -1) @ leaves[2], leaves, dout.double())
    for a, b in zip(got, want):
        for i in (0, 1):
            assert (a[i].double() - b[i]).norm() <= 8 * 2.0 ** -11 * b[i].norm() + 2.0 ** -25 * b[i].numel() ** 0.5, i
    assert ops.train_status() == 0
