"""cswap_b200: B200-native compressed tensor-swap path (ZFP fixed-rate and
zero-value sparse codecs, swap manager, cost model) and operators of a training
step that save little for backward, linear layers on 8-bit floating-point
operands and the optimizer's step, behind a C ABI.

The CUDA library is the only implementation: importing the codec functions
without ``libcswap_b200.so`` raises, there is no CPU path.
"""
from ._lib import lib, LibraryMissing, CswapError, check  # noqa: F401
from .codec import (  # noqa: F401
    POLICY_KEEP, POLICY_DROP, POLICY_RAW, POLICY_SPARSE, POLICY_ZFP, POLICY_Q8,
    zfp_max_bytes, zfp_compress, zfp_decompress, zfp_view,
    sparse_layout, sparse_compress, sparse_decompress, sparse_packed_bytes,
    legacy_sparse_compress, legacy_sparse_decompress,
)
from .swap import SwapManager, Ticket, CostModel, TensorDesc, blob_info  # noqa: F401
from .ops import (  # noqa: F401
    q8_bytes, q8_compress, q8_decompress, gelu_forward, gelu_backward, gelu, gelu_linear,
    layer_norm_forward, layer_norm_backward, layer_norm, attention_forward, attention_backward, attention,
    device_status,
)
from .fp8 import fp8_quantize, fp8_dequantize, fp8_matmul, fp8_linear  # noqa: F401
from .optim import (  # noqa: F401
    AdamW, adamw_step, adamw8_step, adamw8_state, adamw8_pack, adamw8_unpack, gradient_norm,
)
from .execution import Execution, LayerType  # noqa: F401

__version__ = "0.1.0"
