"""What the front ends of the training step's operators share: the native module and types."""
from __future__ import annotations

import ctypes as C
import importlib.util
import threading

import torch

from .. import _build, _lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
NO_TYPE = 9  # what the native module refuses

_lock = threading.Lock()
_module = None


def native():
    """The native module over the loaded library (``HC_CUDA_LIB`` and the instrumented build included)."""
    return _module or _load()


def _load():
    global _module
    with _lock:
        if _module is None:
            lib = _lib.cuda()
            path = _build.build_torch()
            spec = importlib.util.spec_from_file_location("_homcomp_torch", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
            names = ("hc_layer_norm", "hc_layer_norm_backward_bytes", "hc_layer_norm_backward", "hc_token_logprobs", "hc_token_logprobs_backward",
                     "hc_align_rows", "hc_linear_bytes", "hc_linear", "hc_linear_backward_bytes", "hc_linear_backward", "hc_orthogonalize_bytes", "hc_orthogonalize",
                     "hc_adamw", "hc_adamw_values", "hc_linear_cross_entropy_bytes", "hc_linear_cross_entropy", "hc_linear_cross_entropy_backward_bytes",
                     "hc_linear_cross_entropy_backward", "hc_attention_stats", "hc_attention", "hc_attention_backward_bytes", "hc_attention_backward")
            module.bind({name: C.cast(getattr(lib, name), C.c_void_p).value for name in names})
            _module = module
    return _module


def type_code(dtype) -> int:
    """The library's number of a type, -1 for None."""
    return -1 if dtype is None else TYPES.get(dtype, NO_TYPE)


def train_status(device=None, clear: bool = True) -> int:
    """Synchronises and returns the sticky status of the operators' kernels on a device (0 = ok, 3 = a wait ran out)."""
    with torch.cuda.device(device):
        return int(_lib.cuda().hc_train_status(1 if clear else 0))
