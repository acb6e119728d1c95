"""MI355X (gfx950) W4G64 INT4 linear backend for Qwen2 -- HIP kernels behind
the reference's explicit backend selection (src/qwen_int4/backends.py,
src/qwen_int4/linear.py)."""

from .backends import (
    SUPPORTED_BACKENDS,
    hip_w4g64_linear,
    lpu_w4g64_linear,
    torch_w4g64_linear,
    validate_canonical_w4g64_inputs,
)
from .kernels import (
    dequantize_canonical_w4g64_hip,
    hip_available,
    linear_canonical_w4g64_hip,
    linear_kernel_name,
    unpack_canonical_signed_int4_hip,
)
from .linear import QuantLinear
from .packed import packed_attention_hip
from .paged import paged_append_hip, paged_attention_hip, verify_drafts_hip
from .pages import paged_compact_hip, paged_fork_hip, paged_resize_hip
from .quantization import (
    PackingFormat,
    dequantize_groupwise,
    pack_int4,
    quantize_asymmetric_rtn,
    quantize_symmetric_rtn,
    unpack_int4,
)

__all__ = [
    "PackingFormat",
    "QuantLinear",
    "dequantize_groupwise",
    "pack_int4",
    "quantize_asymmetric_rtn",
    "quantize_symmetric_rtn",
    "unpack_int4",
    "SUPPORTED_BACKENDS",
    "dequantize_canonical_w4g64_hip",
    "hip_available",
    "hip_w4g64_linear",
    "lpu_w4g64_linear",
    "torch_w4g64_linear",
    "linear_canonical_w4g64_hip",
    "linear_kernel_name",
    "packed_attention_hip",
    "paged_append_hip",
    "paged_attention_hip",
    "paged_compact_hip",
    "paged_fork_hip",
    "paged_resize_hip",
    "verify_drafts_hip",
    "unpack_canonical_signed_int4_hip",
    "validate_canonical_w4g64_inputs",
]
