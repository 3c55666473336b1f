"""Residual addition, RMS norm and quantisation of its output in one pass (csrc/mtq_mx.hip)."""

from __future__ import annotations

import torch

from ...._ext import ops
from .mx import check_device, format_code, refuse_grad

__all__ = ["rms_norm_quantize"]


def rms_norm_quantize(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    *,
    residual: torch.Tensor | None = None,
    format: str = "mxfp8",
    amax: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """``h = x + residual``; ``y = h * rsqrt(mean(h**2) + eps) * weight``; returns ``(data, scale, h)``.

    ``data`` / ``scale`` are ``y`` in ``format`` (as ``mx_quantize``, what ``mx_linear`` takes with
    ``x_scale``), quantised from the fp32 ``y`` -- the rounding of ``y`` to ``x.dtype`` that a norm which
    stores it makes does not happen (``"fp8_token"``: from the quotients of ``h * weight`` and its maximum, in
    which the root cancels).  ``h`` is the new residual stream, rounded to ``x.dtype`` before the norm
    reads it, as a layer that stores it has it; ``None`` without ``residual``.  ``x [..., H]`` bf16, fp16 or
    fp32, ``H`` at most 65536 and a multiple of 32 for the MX formats; ``weight [H]`` in that dtype or fp32."""
    kind = format_code(format)
    check_device("rms_norm_quantize", x)
    refuse_grad("rms_norm_quantize", x, weight, residual)
    data, scale, h = ops().rms_norm_quantize(x, residual, weight, eps, kind, amax)
    return data, scale, h if residual is not None else None
