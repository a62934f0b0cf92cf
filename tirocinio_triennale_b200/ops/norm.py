"""Layer norm with its backward pass on torch tensors."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._train import TYPES, call, floating, packed, ptr, size, vector, wants_grad


def _forward(x, weight, bias, eps, out_dtype, keep):
    width = x.shape[-1]
    rows = x.numel() // width
    y = torch.empty_like(x, dtype=out_dtype)
    stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if keep else None
    param = weight if weight is not None else bias
    call("layer_norm", "hc_layer_norm", x.device, x.data_ptr(), TYPES[x.dtype], ptr(weight), ptr(bias),
         0 if param is None else TYPES[param.dtype], y.data_ptr(), TYPES[out_dtype], ptr(stats), rows, width, eps)
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, stats = _forward(x, weight, bias, eps, out_dtype, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        width = x.shape[-1]
        rows = x.numel() // width
        dy = packed(dy)
        param = weight if weight is not None else bias
        sums = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        both = torch.empty(2, width, dtype=param.dtype, device=x.device) if sums else None
        need = size("hc_layer_norm_backward_bytes", x.device, rows, width) if sums else 0
        scratch = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        dweight, dbias = (None, None) if both is None else both.unbind(0)
        call("layer_norm backward", "hc_layer_norm_backward", x.device, dy.data_ptr(), TYPES[dy.dtype], x.data_ptr(),
             TYPES[x.dtype], ptr(weight), 0 if param is None else TYPES[param.dtype], stats.data_ptr(), ptr(dx), ptr(dweight),
             ptr(dbias), rows, width, ptr(scratch), need)
        return (dx, dweight if ctx.needs_input_grad[1] else None, dbias if ctx.needs_input_grad[2] else None, None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, with gradients of ``x``, ``weight`` and ``bias``.

    ``x``: float32, bfloat16 or float16, any shape; ``weight`` and ``bias``: one value per column, both of one of these types.
    The result has ``x``'s type, or ``out_dtype``: a float32 residual stream can give bfloat16 rows to a product, which saves a
    conversion.  Of the two 16-bit types one call takes only one.  Statistics and sums are held in float32; the sums of the
    gradients of ``weight`` and ``bias`` are formed in a fixed order.  Tensors with gaps are copied."""
    floating("x", x)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm: x has no columns")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in TYPES or (torch.float32 not in (x.dtype, out_dtype) and x.dtype != out_dtype):
        raise ValueError("layer_norm: no %s result of %s rows" % (out_dtype, x.dtype))
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            vector(name, t, x.shape[-1], x.device)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("layer_norm: weight and bias have different types")
    if not eps >= 0:
        raise ValueError("layer_norm: eps is negative")
    x = packed(x)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps), out_dtype)
    return _forward(x, weight, bias, float(eps), out_dtype, False)[0]
