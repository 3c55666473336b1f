"""``mtq.compress``: pack the weights of a quantized model into real-quantized QTensors
(reference quantization/compress.py:53-227).

Every QuantLinear whose weight quantizer matches the compress config gets ``fake_quant=False``
and its weight replaced by a ``QTensorWrapper`` (FP8 / INT8 / INT4 / NVFP4 / MXFP4 / MXFP8), the
scales kept as ``_scale`` / ``_double_scale`` buffers of the weight quantizer; the module becomes
a ``RealQuantLinear`` whose forward dequantises the packed weight (the reference's fallback when
no real-quant GEMM backend matches).  With ``"mx_gemm": True`` it multiplies with the packed weight where
the format has a product here: MXFP4 weights behind an MXFP4, MXFP8 or per-tensor FP8 input quantizer
(``MXFP4_DEFAULT_CFG``, ``W4A8_MXFP4_FP8_CFG``), ``kernels.quantization.mx_linear``.  The packing runs on
the MI355X export kernels where the format has one (qtensor/__init__.py).
"""

from __future__ import annotations

import fnmatch
import warnings
from typing import Any

import torch
import torch.nn as nn

from ..kernels.quantization import mx_linear
from ..kernels.quantization.mx import needs_grad
from .conversion import set_quantizer_attributes_partial
from .nn.modules.quant_linear import _QuantLinear
from .nn.modules.tensor_quantizer import TensorQuantizer
from .qtensor import MXFP4QTensor, QTensorWrapper, pack_real_quantize_weight
from .utils.names import is_quantized_linear

__all__ = ["CompressConfig", "RealQuantLinear", "compress", "is_real_quantized"]


class CompressConfig(dict):
    """{"compress": {pattern: bool}, "quant_gemm": bool} (reference config.py:1620-1633), and ``"mx_gemm"``:
    multiply packed MXFP4 weights as they are (``RealQuantLinear``) instead of dequantising them.  Off unless
    asked for: the outputs differ from the dequantised ones in their last bits."""

    def __init__(self, compress: dict[str, bool] | None = None, quant_gemm: bool = True, mx_gemm: bool = False):
        super().__init__(compress=dict(compress) if compress is not None else {"*": True}, quant_gemm=quant_gemm)
        if mx_gemm:
            self["mx_gemm"] = True

    @property
    def compress(self) -> dict[str, bool]:
        return self["compress"]

    @property
    def quant_gemm(self) -> bool:
        return self["quant_gemm"]

    @property
    def mx_gemm(self) -> bool:
        return self.get("mx_gemm", False)


def _runs_more_than_its_forward(module) -> bool:
    """Whether a call of ``module`` does more than its class's forward: hooks of its own or of every module, a
    forward put in its place."""
    hooks = torch.nn.modules.module
    return bool(
        module._forward_hooks or module._forward_pre_hooks or hooks._global_forward_hooks or hooks._global_forward_pre_hooks
        or "forward" in module.__dict__
    )


def _mx_gemm_format(module, input):
    """``(format, amax)`` when ``module``'s forward on ``input`` is ``mx_linear`` of its packed weight: an
    MXFP4 weight with the input's dtype, an input quantizer that only fake-quantises to a format
    ``mx_linear`` takes, no gradient, nothing hooked to the quantizers' calls, which do not happen; else None."""
    weight = module._parameters.get("weight")
    if not isinstance(weight, QTensorWrapper) or weight.metadata["qtensor_class"] is not MXFP4QTensor:
        return None
    if not isinstance(input, torch.Tensor) or not input.is_cuda or input.dtype != weight.metadata["dtype"]:
        return None
    if input.dtype not in (torch.bfloat16, torch.float16, torch.float32) or weight.device != input.device:
        return None
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") != input.dtype:
        return None  # the linear's output would have the autocast dtype
    wq, iq = module._modules.get("weight_quantizer"), module._modules.get("input_quantizer")
    if type(wq) is not TensorQuantizer or type(iq) is not TensorQuantizer:
        return None
    if _runs_more_than_its_forward(wq) or _runs_more_than_its_forward(iq):
        return None
    if not wq.is_enabled or not wq._if_quant or wq._if_calib or not wq.is_mxfp(4) or wq.pre_quant_scale is not None:
        return None
    n, k = weight.metadata["shape"]
    scale = getattr(wq, "_scale", None)
    if scale is None or scale.dtype != torch.uint8 or k % 32 or scale.numel() * 32 != n * k or input.shape[-1] != k:
        return None
    bias = module._parameters.get("bias")
    if bias is not None and bias.dtype not in (input.dtype, torch.float32):
        return None
    if needs_grad(input, bias):
        return None
    if not iq.is_enabled or not iq._if_quant or iq._if_calib or not iq._fake_quant:
        return None
    if iq.backend is not None or iq.pre_quant_scale is not None or iq.rotate_is_enabled or iq.bias is not None:
        return None
    if iq.is_mxfp(4):
        return "mxfp4", None
    if iq.is_mxfp(8):
        return "mxfp8", None
    if iq.is_fp8 and not iq._dynamic:
        amax = iq._get_amax(input)  # calibrated, or the input's own
        if amax.numel() == 1:
            return "fp8", amax.to(torch.float32).reshape(1)
    return None


class RealQuantLinear(_QuantLinear):
    """QuantLinear with a packed weight (reference nn/modules/quant_linear.py:196-300).  Without a
    real-quant GEMM the forward is the fake-quant one, whose weight quantizer dequantises.

    With ``mx_gemm`` and a format that has one (``_mx_gemm_format``) the input is quantised by the same rules to its codes and multiplied
    by the weight's, so the result differs from the fallback's by its sums (``mx_linear`` says how far), and
    for a per-tensor FP8 input by the rounding of the dequantised input to its dtype that no longer happens."""

    list_of_scale_tensors = ["_scale", "_double_scale", "_scale_zeros"]
    allow_real_quant_gemm = True

    def forward(self, input, *args, **kwargs):
        if getattr(self, "_use_mx_gemm", False) and not args and not kwargs:
            gemm = _mx_gemm_format(self, input)
            if gemm is not None:
                fmt, amax = gemm
                y = mx_linear(input, self._parameters["weight"].data, self.weight_quantizer._scale,
                              self._parameters.get("bias"), format=fmt, amax=amax)
                return self.output_quantizer(y)
        if getattr(self, "_use_real_quant_gemm", False) and not self.__dict__.get("_warned_no_gemm"):
            warnings.warn(f"RealQuantLinear: No real-quant GEMM found: {type(self).__name__}.")
            self.__dict__["_warned_no_gemm"] = True
        return super().forward(input, *args, **kwargs)


def _to_real_quant_class(module: nn.Module) -> None:
    if isinstance(module, RealQuantLinear):
        return
    orig = module._original_cls
    module.__class__ = type(f"RealQuant{orig.__name__}", (RealQuantLinear, orig), {"_original_cls": orig})


def _as_config(config) -> CompressConfig:
    if config is None:
        return CompressConfig()
    if isinstance(config, CompressConfig):
        return config
    if isinstance(config, dict) and ("compress" in config or "quant_gemm" in config or "mx_gemm" in config):
        return CompressConfig(config.get("compress"), config.get("quant_gemm", True), config.get("mx_gemm", False))
    if isinstance(config, dict):
        return CompressConfig(config)
    raise TypeError(f"Invalid compress config {config!r}")


def compress_convert(model: nn.Module, config: CompressConfig, skip_real_quantize_weight: bool = False):
    """reference compress.py:53-133."""
    for _, module in model.named_modules():
        if is_quantized_linear(module) and isinstance(module, _QuantLinear):
            _to_real_quant_class(module)
    cfg = config.compress
    if "default" in cfg and isinstance(cfg["default"], bool):
        set_quantizer_attributes_partial(model, "*weight_quantizer*", {"fake_quant": not cfg["default"]})
    for pattern, to_compress in cfg.items():
        if pattern == "default":
            continue
        if not isinstance(to_compress, bool):
            raise ValueError(f"Invalid compression configuration: {to_compress}, expected a boolean as value.")
        set_quantizer_attributes_partial(
            model, lambda name, p=pattern: fnmatch.fnmatch(name, p) and "weight_quantizer" in name,
            {"fake_quant": not to_compress},
        )
    if not skip_real_quantize_weight:
        pack_real_quantize_weight(model)
    if any(isinstance(getattr(m, "weight", None), QTensorWrapper) for m in model.modules()):
        warnings.warn(
            "Real quantization has been applied to the model. This feature is still experimental, "
            "and some functionalities may not be supported."
        )
    for m in model.modules():
        if isinstance(m, RealQuantLinear):
            m._use_real_quant_gemm = bool(config.quant_gemm) and m.allow_real_quant_gemm
            m._use_mx_gemm = config.mx_gemm and m._use_real_quant_gemm
    metadata: dict[str, Any] = {"real_quantizer_state": {}, "q_tensor_state": {}}
    for name, m in model.named_modules():
        if isinstance(m, RealQuantLinear):
            metadata["real_quantizer_state"][name] = m.weight_quantizer.get_modelopt_state()
            if isinstance(m.weight, QTensorWrapper):
                metadata["q_tensor_state"][name] = m.weight.get_state()
    return model, metadata


def compress(model: nn.Module, config=None) -> None:
    """Compress the weights of a quantized model in place (reference compress.py:196-221)."""
    cfg = _as_config(config)
    with torch.no_grad():
        _, metadata = compress_convert(model, cfg)
    entry = model.__dict__.setdefault("_modelopt_amd_mode", {"config": {}})
    entry["compress"] = {"config": dict(cfg), "metadata": metadata}


def is_real_quantized(model: nn.Module) -> bool:
    return any(isinstance(m, RealQuantLinear) for m in model.modules())
