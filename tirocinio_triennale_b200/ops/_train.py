"""What the front ends of the training step's operators share: types, checks of tensors, calls."""
from __future__ import annotations

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


def call(what: str, name: str, device: torch.device, *args):
    """The native function on the current stream of ``device``, with that device current."""
    fn = getattr(_lib.cuda(), name)
    index = device.index
    if _current_device() == index:
        st = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _raw_stream(index))
    if st:
        _lib.check(st, what)


def size(name: str, device: torch.device, *args) -> int:
    """A native function that says how much scratch memory a call needs."""
    if _current_device() == device.index:
        return getattr(_lib.cuda(), name)(*args)
    with torch.cuda.device(device):
        return getattr(_lib.cuda(), name)(*args)


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
