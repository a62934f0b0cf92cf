"""Signatures of the training step's operators in libhomcomp_b200.so (csrc/include/homcomp_train.h)."""
from __future__ import annotations

import ctypes as C

vp = C.c_void_p


def declare(lib):
    sz, f, i, l = C.c_size_t, C.c_float, C.c_int, C.c_int64
    sizes = {
        "hc_layer_norm_backward_bytes": [sz, sz],
        "hc_linear_bytes": [sz, sz, sz],
        "hc_linear_backward_bytes": [sz, sz, sz, i],
        "hc_orthogonalize_bytes": [sz, sz, sz],
    }
    sigs = {
        "hc_layer_norm": [vp, i, vp, vp, i, vp, i, vp, sz, sz, f, vp],
        "hc_layer_norm_backward": [vp, i, vp, i, vp, i, vp, vp, vp, vp, sz, sz, vp, sz, vp],
        "hc_align_rows": [vp, sz, sz, sz, vp, sz, vp],
        "hc_linear": [vp, sz, vp, sz, i, vp, i, vp, sz, vp, i, sz, vp, sz, i, sz, sz, sz, vp, sz, vp],
        "hc_linear_backward": [vp, i, sz, vp, sz, i, i, vp, sz, vp, sz, i, vp, sz, vp, sz, vp, i, sz, sz, sz, vp, sz, vp],
        "hc_orthogonalize": [vp, i, sz, sz, sz, sz, sz, vp, i, f, f, f, f, vp, sz, vp],
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
