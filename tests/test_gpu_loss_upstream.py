"""Rows that ``ignore_index`` leaves out of a loss have a gradient of 0, whatever comes from upstream."""
import math

import pytest
import torch

from tirocinio_triennale_b200 import ops

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("upstream", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_rows_left_out_have_no_part_of_an_upstream_gradient_that_is_no_number(reduction, upstream, kind):
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(40, 24, generator=g).to(kind).cuda().requires_grad_(), torch.randn(50, 24, generator=g).to(kind).cuda().requires_grad_()
    t = torch.randint(0, 50, (40,), generator=g).cuda()
    t[::3] = -100
    loss = ops.linear_cross_entropy(x, w, t, reduction=reduction)
    (dx,) = torch.autograd.grad(loss, x, torch.full_like(loss, upstream))
    assert (dx[::3] == 0).all() and not dx[1::3].isfinite().any()  # a sum that is finite times an infinity is one
    # nobody has a token
    loss = ops.linear_cross_entropy(x, w, torch.full_like(t, -100), reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), torch.full_like(loss, upstream))
    assert (dx == 0).all() and (dw == 0).all()
