"""What the front ends of the training step's operators share: types, checks of tensors, calls."""
from __future__ import annotations

import functools

import torch

from .. import _lib
from .codec import _current_device, _raw_stream

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def floating(name: str, t: torch.Tensor, device=None):
    """``t`` is a CUDA tensor of one of the three types, on ``device`` where that is given."""
    if not isinstance(t, torch.Tensor) or t.dtype not in TYPES:
        raise ValueError("%s: expected a float32, bfloat16 or float16 tensor" % name)
    if not t.is_cuda:
        raise ValueError("%s: expected a CUDA tensor" % name)
    if device is not None and t.device != device:
        raise ValueError("%s is on %s, not on %s" % (name, t.device, device))


def vector(name: str, t: torch.Tensor, n: int, device):
    floating(name, t, device)
    if t.shape != (n,):
        raise ValueError("%s: expected %d values in one dimension, got shape %s" % (name, n, tuple(t.shape)))


def packed(t: torch.Tensor) -> torch.Tensor:
    """``t`` without gaps and 16-byte aligned, copied only if it is not."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def ptr(t):
    return None if t is None else t.data_ptr()


_functions = {}  # native functions by name


def _function(name: str):
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(_lib.cuda(), name)
    return fn


def call(what: str, name: str, device: torch.device, *args):
    """The native function on the current stream of ``device``, with that device current."""
    fn = _functions.get(name) or _function(name)
    index = device.index
    if _current_device() == index:
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _raw_stream(index))
    if st:
        _lib.check(st, what)


@functools.lru_cache(maxsize=4096)
def _size(name: str, index: int, *args) -> int:
    with torch.cuda.device(index):
        return _function(name)(*args)


def size(name: str, device: torch.device, *args) -> int:
    """A native function that says how much scratch memory a call needs: it goes by sizes and the device alone."""
    return _size(name, device.index, *args)


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def train_status(device=None, clear: bool = True) -> int:
    """Synchronises and returns the sticky status of the products' kernels on a device (0 = ok, 3 = a wait ran out)."""
    with torch.cuda.device(device):
        torch.cuda.synchronize()
        return int(_lib.cuda().hc_train_status(1 if clear else 0))


def padded(n: int) -> int:
    return (n + 7) // 8 * 8


def empty_rows(rows: int, width: int, dtype, device) -> torch.Tensor:
    """A matrix whose rows begin at 16-byte boundaries: with gaps where eight does not divide ``width``."""
    t = torch.empty(rows, padded(width), dtype=dtype, device=device)
    return t if t.shape[1] == width else t[:, :width]


def any_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else padded(t.shape[1])


def rows_adjacent(t: torch.Tensor) -> bool:
    """A matrix whose rows' elements are adjacent and whose rows do not overlap."""
    return (t.stride(1) == 1 or t.shape[1] == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])


def is_operand(t: torch.Tensor) -> bool:
    """A matrix as the products read it: rows of adjacent elements that begin at 16-byte boundaries."""
    return rows_adjacent(t) and row_stride(t) % 8 == 0 and t.data_ptr() % 16 == 0


def operand(t: torch.Tensor) -> torch.Tensor:
    return t if is_operand(t) else empty_rows(t.shape[0], t.shape[1], t.dtype, t.device).copy_(t)
