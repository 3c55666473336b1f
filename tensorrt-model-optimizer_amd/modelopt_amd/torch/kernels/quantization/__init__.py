"""Computing with packed low-bit operands: rows quantised to microscaled (MX) or FP8 formats, the RMS norm
that hands its output over quantised, and the product with packed MXFP4 weights (the reference's
counterparts are its real-quant GEMM backends, modelopt/torch/quantization/backends)."""

from .mx import FORMATS, mx_linear, mx_quantize
from .rms_norm import rms_norm_quantize

__all__ = ["FORMATS", "mx_linear", "mx_quantize", "rms_norm_quantize"]
