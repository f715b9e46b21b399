"""Linear on microscaled 4-bit floats (MXFP4 weight, activations encoded on every forward): the
layer that ``backends.quantized.engine = "mxfp4"`` makes ``convert`` and ``quantize_dynamic`` build.  No
counterpart in the reference; the constructor and ``from_float`` follow ``QuantizedLinearMLX``."""

from __future__ import annotations

import torch

from ... import _lib
from ...quantization._mx import _scale_shape, mx_linear, mx_quantize


class MXLinear(torch.nn.Module):
    def __init__(self, in_features: int, out_features: int, bias: bool = True, relu: bool = False) -> None:
        super().__init__()
        if in_features <= 0 or in_features % 32 != 0:
            raise _lib.ShapeMismatch(f"in_features must be a multiple of 32, got {in_features}")
        self.in_features, self.out_features, self.relu = in_features, out_features, relu
        self.register_buffer("weight_codes", torch.zeros((out_features, in_features // 2), dtype=torch.uint8))
        self.register_buffer("weight_scales", torch.zeros(_scale_shape(out_features, in_features), dtype=torch.uint8))
        if bias:
            self.register_buffer("bias", torch.zeros(out_features))
        else:
            self.bias = None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        _lib.require_cuda(x, "input")
        _lib.check_device_status_lazily(x.device)
        xin = x if x.dtype in (torch.float32, torch.bfloat16) else x.to(torch.float32)
        return mx_linear(xin, self.weight_codes, self.weight_scales, bias=self.bias, relu=self.relu)

    @classmethod
    def from_float(cls, mod: torch.nn.Module, relu: bool = False) -> "MXLinear":
        m = cls(mod.in_features, mod.out_features, bias=mod.bias is not None, relu=relu)
        w = mod.weight.detach()
        w = w if w.dtype in (torch.float32, torch.bfloat16) else w.to(torch.float32)
        m.weight_codes, m.weight_scales = mx_quantize(w)
        if mod.bias is not None:
            m.bias = mod.bias.detach().to(torch.float32)
        return m

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, relu={self.relu}, format=mxfp4"
