"""Matrix product with bias, activation and residual in its epilogue, and its backward pass."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._train import (TYPES, any_stride, call, empty_rows, floating, is_operand, operand, padded, ptr, row_stride, rows_adjacent, size, vector,
                     wants_grad)

ACTIVATIONS = {None: 0, "gelu_tanh": 1, "relu": 2, "silu": 3}
FEW_ROWS = 8  # up to here W is read by a kernel that takes rows that begin anywhere


def _forward(x, weight, bias, residual, act, out_dtype, keep):
    m, k = x.shape
    n = weight.shape[0]
    dev = x.device
    out = empty_rows(m, n, out_dtype, dev)
    z = empty_rows(m, n, x.dtype, dev) if keep and act else None
    call("linear", "hc_linear", dev, x.data_ptr(), row_stride(x), weight.data_ptr(), row_stride(weight), TYPES[x.dtype], ptr(bias),
         0 if bias is None else TYPES[bias.dtype], ptr(residual), 0 if residual is None else any_stride(residual), out.data_ptr(),
         TYPES[out_dtype], padded(n), ptr(z), padded(n), act, m, k, n)
    return out, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_dtype):
        out, z = _forward(x, weight, bias, residual, act, out_dtype, True)
        ctx.save_for_backward(x, weight, z)
        ctx.act = act
        ctx.bias_dtype = None if bias is None else bias.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        (m, k), n, dev, t = x.shape, weight.shape[0], x.device, x.dtype
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        if not (want_x or want_w or want_b):
            return None, None, None, dy if want_r else None, None, None
        g = dy if rows_adjacent(dy) else dy.contiguous()
        # dz is written where dy itself is not what the products can read
        keep = 1 if ctx.act or dy.dtype != t or not is_operand(g) else 0
        dx = empty_rows(m, k, t, dev) if want_x else None
        dw = empty_rows(n, k, t, dev) if want_w else None
        db = torch.empty(n, dtype=ctx.bias_dtype, device=dev) if want_b else None
        w = operand(weight) if want_x else weight
        a = operand(x) if want_w else x
        need = size("hc_linear_backward_bytes", dev, m, k, n, keep) if m else 0
        scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        call("linear backward", "hc_linear_backward", dev, g.data_ptr(), TYPES[g.dtype], any_stride(g), ptr(z), padded(n), ctx.act, keep,
             a.data_ptr(), row_stride(a), w.data_ptr(), row_stride(w), TYPES[t], ptr(dx), padded(k), ptr(dw), padded(k), ptr(db),
             0 if db is None else TYPES[db.dtype], m, k, n, ptr(scratch), need)
        return dx, dw, db, dy if want_r else None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None,
           residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` with gradients of all four tensors.

    ``x`` (..., inner) and ``weight`` (width, inner): both bfloat16 or both float16, products summed in float32.  ``bias``: one value
    per column, of any of the three types.  ``activation``: None, "gelu_tanh", "relu" or "silu".  ``residual``: of the result's shape,
    float32 or ``x``'s type, and the result has its type; without one the result has ``x``'s type or ``out_dtype`` (float32).

    Everything behind the product happens before the result is stored.  For the backward pass of an activation its argument is
    kept in ``x``'s type, and the gradient is rounded to that type before it enters the products; gradients of ``x`` and ``weight``
    have their types, that of ``bias`` its own, summed in float32 in a fixed order.  Where eight does not divide ``width`` the
    result's rows are kept apart so that they begin at 16-byte boundaries: it is a view with gaps."""
    floating("x", x)
    floating("weight", weight, x.device)
    if x.dtype == torch.float32 or weight.dtype != x.dtype:
        raise ValueError("linear: x and weight are both bfloat16 or both float16, got %s and %s" % (x.dtype, weight.dtype))
    if x.dim() == 0 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError("linear: no product of x %s and weight %s" % (tuple(x.shape), tuple(weight.shape)))
    if activation not in ACTIVATIONS:
        raise ValueError("linear: activation is one of %s" % ", ".join(map(str, ACTIVATIONS)))
    n, k = weight.shape
    if bias is not None:
        vector("bias", bias, n, x.device)
        bias = bias.contiguous()
    shape = (*x.shape[:-1], n)
    if residual is not None:
        floating("residual", residual, x.device)
        if residual.shape != shape:
            raise ValueError("linear: residual has shape %s, the result %s" % (tuple(residual.shape), shape))
        if out_dtype is not None and out_dtype != residual.dtype:
            raise ValueError("linear: the result has the residual's type")
        out_dtype = residual.dtype
        residual = residual.reshape(-1, n)
        residual = residual if rows_adjacent(residual) else residual.contiguous()
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in (torch.float32, x.dtype):
        raise ValueError("linear: the result is float32 or of x's type")
    flat = x.reshape(-1, k)
    if max(flat.shape[0], n, k) >= 1 << 26:
        raise ValueError("linear: every side is below 2^26")
    if flat.shape[0] > FEW_ROWS:
        flat, weight = operand(flat), operand(weight)
    else:
        flat = flat if rows_adjacent(flat) else flat.contiguous()
        weight = weight if rows_adjacent(weight) else weight.contiguous()
    act = ACTIVATIONS[activation]
    if wants_grad(flat, weight, bias, residual):
        out = _Linear.apply(flat, weight, bias, residual, act, out_dtype)
    else:
        out = _forward(flat, weight, bias, residual, act, out_dtype, False)[0]
    return out if len(shape) == 2 else out.reshape(shape)
