"""Signatures of the training step's operators in libhomcomp_b200.so (csrc/include/homcomp_train.h)."""
from __future__ import annotations

import ctypes as C

vp = C.c_void_p


class Heads(C.Structure):
    """hc_heads: a tensor of (batch, head, position, value) with its strides."""

    _fields_ = [("data", C.c_void_p), ("batch", C.c_size_t), ("head", C.c_size_t), ("position", C.c_size_t)]


def declare(lib):
    sz, f, d, i, l = C.c_size_t, C.c_float, C.c_double, C.c_int, C.c_int64
    sizes = {
        "hc_layer_norm_backward_bytes": [sz, sz],
        "hc_linear_bytes": [sz, sz, sz],
        "hc_linear_backward_bytes": [sz, sz, sz, i],
        "hc_orthogonalize_bytes": [sz, sz, sz],
        "hc_attention_stats": [sz, sz, sz],
        "hc_attention_backward_bytes": [sz] * 6,
        "hc_linear_cross_entropy_bytes": [sz, sz, sz],
        "hc_linear_cross_entropy_backward_bytes": [sz, sz, sz],
    }
    sigs = {
        "hc_layer_norm": [vp, i, vp, vp, i, vp, i, vp, sz, sz, f, vp],
        "hc_layer_norm_backward": [vp, i, vp, i, vp, i, vp, vp, vp, vp, sz, sz, vp, sz, vp],
        "hc_align_rows": [vp, sz, sz, sz, vp, sz, vp],
        "hc_linear": [vp, sz, vp, sz, i, vp, i, vp, sz, vp, i, sz, vp, sz, i, sz, sz, sz, vp, sz, vp],
        "hc_linear_backward": [vp, i, sz, vp, sz, i, i, vp, sz, vp, sz, i, vp, sz, vp, sz, vp, i, sz, sz, sz, vp, sz, vp],
        "hc_orthogonalize": [vp, i, sz, sz, sz, sz, sz, vp, i, f, f, f, f, vp, sz, vp],
        "hc_attention": [Heads, Heads, Heads, i, vp, vp, sz, sz, sz, sz, sz, sz, sz, sz, f, vp],
        "hc_attention_backward": [Heads, vp, Heads, Heads, Heads, i, vp, vp, vp, vp, sz, sz, sz, sz, sz, sz, sz, sz, f, vp, sz, vp],
        "hc_linear_cross_entropy": [vp, sz, vp, sz, i, vp, l, i, vp, vp, sz, sz, sz, vp, sz, vp],
        "hc_linear_cross_entropy_backward": [vp, sz, vp, sz, i, vp, l, i, vp, vp, vp, sz, vp, sz, sz, sz, sz, vp, sz, vp],
        "hc_adamw": [vp, sz, i, i, i, d, vp, d, d, d, d, l, vp, C.c_uint64, vp],
        "hc_adamw_values": [vp, vp, vp, sz, vp, vp, vp],
        "hc_train_status": [i],
        "hc_token_logprobs": [vp, i, sz, sz, sz, vp, l, i, vp, vp, vp, vp, vp, vp],
        "hc_token_logprobs_backward": [vp, i, sz, sz, sz, vp, l, vp, vp, vp, vp, sz, vp],
    }
    for names, restype in ((sizes, sz), (sigs, i)):
        for name, args in names.items():
            fn = getattr(lib, name, None)
            if fn is not None:
                fn.restype = restype
                fn.argtypes = args
