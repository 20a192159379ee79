"""A linear layer on 4-bit weights (the inference form of ``_YvQuantizedLinear``,
model/utils/quantization.py:412-496, with group scales)."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import functional as yvf
from .checkpoint import StateSource, linear_weight
from .quant import PackedLinear, pack_linear

_GROUP = 128


class YvInt4Linear(nn.Module):
    """y = x Wᵀ + b with W in int4 and a bf16 scale per 128 columns of a row (quant.pack_linear).

    forward(x [..., in_features]) -> [..., out_features] in x's dtype (bfloat16 or float32), for any
    number of rows. Inference only: no gradients, and a forward in training mode raises. ``codes`` and
    ``scales`` are buffers, so that ``state_dict``, ``to(device)`` and ``load_state_dict`` take them
    along; scales are held as int16, the bits of their bf16 values, so that a change of the module's
    dtype leaves them as they are (the bias follows it).
    """

    def __init__(self, in_features: int, out_features: int, bias: bool = True, device=None, dtype=None):
        super().__init__()
        if in_features < 1 or out_features < 1:
            raise ValueError(f"a linear layer needs features, got in {in_features}, out {out_features}")
        self.in_features, self.out_features = in_features, out_features
        blocks, groups = -(-out_features // 16), -(-in_features // _GROUP)
        self.register_buffer("codes", torch.full((blocks, groups, 1024), 0x88, dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.zeros(blocks, groups, 16, dtype=torch.int16, device=device))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype), requires_grad=False)
        else:
            self.register_parameter("bias", None)

    @classmethod
    def from_linear(cls, linear: nn.Linear, dtype=None) -> "YvInt4Linear":
        """A packed copy of ``linear`` on its device; ``dtype`` of the bias (its own when None)."""
        w = linear.weight.detach()
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, w.device,
                w.dtype if dtype is None else dtype)
        m.set_weight(pack_linear(w.float()))
        if linear.bias is not None:
            m.bias.copy_(linear.bias.detach())
        return m.eval()

    @property
    def packed(self) -> PackedLinear:
        return PackedLinear(self.in_features, self.out_features, self.codes, self.scales.view(torch.bfloat16))

    def set_weight(self, packed: PackedLinear) -> None:
        """Takes over packed weights (onto the module's device)."""
        if (packed.in_features, packed.out_features) != (self.in_features, self.out_features):
            raise ValueError(f"packed weight is {packed.out_features} x {packed.in_features}, "
                             f"the layer {self.out_features} x {self.in_features}")
        self.codes = packed.codes.to(self.codes.device)
        self.scales = packed.scales.to(self.scales.device).view(torch.int16)

    def load_reference_state_dict(self, src, name: str) -> None:
        """The Linear ``name`` of a reference state dict, full precision or quantized
        (``checkpoint.linear_weight``), packed, and its ``bias``, which the checkpoint has if and only if the
        layer does."""
        key = f"{name}.bias"
        if self.bias is not None and key not in src:
            raise KeyError(f"{key}: not in the checkpoint")
        if self.bias is None and key in src:
            raise ValueError(f"{key}: the layer has no bias")
        self.set_weight(pack_linear(linear_weight(src, name).to(self.codes.device)))
        if self.bias is not None:
            with torch.no_grad():
                self.bias.copy_(src.get(key) if isinstance(src, StateSource) else src[key])

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.training:
            raise NotImplementedError("YvInt4Linear is an inference forward; call .eval()")
        if not x.is_contiguous():
            x = x.contiguous()
        return yvf.int4_linear(x, self.packed, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
