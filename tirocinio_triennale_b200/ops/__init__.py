from .cpu_codec import (  # noqa: F401
    cpu_compress, cpu_decompress, cpu_decode_quant, cpu_hom_add, cpu_hom_add_deltas, cpu_hom_add_streams,
    cpu_quant_pred, cpu_quantize, cpu_dequantize, cpu_ring_allreduce, cpu_stream_size, max_compressed_bytes,
    rate_bytes, chunk_elems,
)
from .codec import Codec  # noqa: F401
from . import stream_io  # noqa: F401
from .norm import layer_norm  # noqa: F401
from .logprobs import TokenLogprobs, token_logprobs  # noqa: F401
from .linear import linear  # noqa: F401
from .orthogonalize import orthogonalize  # noqa: F401
from .attention import attention  # noqa: F401
from .loss import linear_cross_entropy  # noqa: F401
from .adamw import adamw_step, adamw_values  # noqa: F401
from ._train import train_status  # noqa: F401
