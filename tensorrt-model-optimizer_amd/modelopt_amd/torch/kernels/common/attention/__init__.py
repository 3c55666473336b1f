"""Flash attention with softmax-P quant-dequant on MFMA (reference
``modelopt/torch/kernels/common/attention``: ``triton_fa.attention`` and the HF wrapper
``hf_triton_attention``), and a paged KV cache in NVFP4 with its attention.  The names of the reference are
kept as aliases."""

from .flash_attention import LOG2E, attention
from .fp4_cache import NVFP4KVCache
from .hf_attention import (
    attention_forward,
    triton_attention_forward,
    validate_attention_envelope,
    validate_triton_attention_envelope,
)

__all__ = [
    "LOG2E",
    "NVFP4KVCache",
    "attention",
    "attention_forward",
    "triton_attention_forward",
    "validate_attention_envelope",
    "validate_triton_attention_envelope",
]
