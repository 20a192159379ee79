"""The gated feed-forward block, dense: one expert of the MoE layer by itself (YvSwiGLUExpert,
model/moe/expert.py:384-489), to be trained in bf16 or fp32 and to be served in 8-bit floating point."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from . import functional as yvf
from .linear import YvFp8Linear
from .quant import PackedExperts, PackedFp8Linear


class YvSwiGLU(nn.Module):
    """down_proj(silu(gate_proj(x)) * up_proj(x)) with gradients (functional.swiglu).

    The parameters have the names and shapes of YvSwiGLUExpert's (``gate_proj.weight``, ``up_proj.weight`` [ffn,
    hidden], ``down_proj.weight`` [hidden, ffn], no biases), so a state dict of an expert loads as it is, and
    quant.pack_experts takes the weights. forward(x [..., hidden]) in the parameters' dtype, bfloat16 or float32, in
    training and in eval mode; torch.autocast casts neither x nor the parameters, and another dtype of x raises.
    """

    def __init__(self, hidden_size: int, intermediate_size: int, device=None, dtype=None):
        super().__init__()
        if hidden_size < 1 or intermediate_size < 1:
            raise ValueError(f"a gated block needs features, got hidden {hidden_size}, ffn {intermediate_size}")
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        kw = dict(bias=False, device=device, dtype=dtype)
        self.gate_proj = nn.Linear(hidden_size, intermediate_size, **kw)
        self.up_proj = nn.Linear(hidden_size, intermediate_size, **kw)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, **kw)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return yvf.swiglu(x.contiguous(), self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight)


class YvFp8SwiGLU(nn.Module):
    """The block on 8-bit weights (functional.fp8_swiglu): YvFp8Linear's buffers under the block's names.

    forward(x [..., hidden] bfloat16) -> bfloat16. Inference only: a forward in training mode raises.
    """

    def __init__(self, hidden_size: int, intermediate_size: int, device=None):
        super().__init__()
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        self.gate_proj = YvFp8Linear(hidden_size, intermediate_size, bias=False, device=device)
        self.up_proj = YvFp8Linear(hidden_size, intermediate_size, bias=False, device=device)
        self.down_proj = YvFp8Linear(intermediate_size, hidden_size, bias=False, device=device)

    @classmethod
    def from_block(cls, block: nn.Module) -> "YvFp8SwiGLU":
        """A packed copy of a block with gate_proj, up_proj and down_proj, without biases (YvSwiGLU, an expert), on its
        device."""
        ffn, hidden = block.gate_proj.weight.shape
        m = cls(hidden, ffn, block.gate_proj.weight.device)
        for name in ("gate_proj", "up_proj", "down_proj"):
            linear = getattr(block, name)
            if linear.bias is not None:
                raise ValueError(f"{name} has a bias: the block has none")
            p = getattr(m, name)
            if (linear.in_features, linear.out_features) != (p.in_features, p.out_features):
                raise ValueError(f"{name} is {linear.out_features} x {linear.in_features}: no gated block of hidden "
                                 f"{hidden}, ffn {ffn}")
            setattr(m, name, YvFp8Linear.from_linear(linear))
        return m.eval()

    @classmethod
    def from_packed_expert(cls, experts: PackedExperts, index: int) -> "YvFp8SwiGLU":
        """Expert ``index`` (routed first, then shared) of an fp8 stack as a block on the same memory."""
        if experts.format != _lib.W_FP8:
            raise ValueError("the experts are not packed in fp8")
        if not 0 <= index < experts.num_total:
            raise ValueError(f"expert {index} of {experts.num_total}")
        H, F = experts.hidden, experts.ffn
        m = cls(H, F, "meta")
        for name, w, s, i, o in (("gate_proj", experts.w_gate, experts.s_gate, H, F),
                                 ("up_proj", experts.w_up, experts.s_up, H, F),
                                 ("down_proj", experts.w_down, experts.s_down, F, H)):
            p = getattr(m, name)
            p.codes = w[index].view(o // 16, i // 128, 2048)
            p.scales = s[index].view(torch.int32)
        return m.eval()

    def load_reference_state_dict(self, src, prefix: str) -> None:
        """The expert under ``prefix`` (ending in a dot, or empty) of a reference state dict, packed."""
        for name in ("gate_proj", "up_proj", "down_proj"):
            getattr(self, name).load_reference_state_dict(src, prefix + name)

    def packed(self) -> tuple[PackedFp8Linear, PackedFp8Linear, PackedFp8Linear]:
        return self.gate_proj.packed, self.up_proj.packed, self.down_proj.packed

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.training:
            raise NotImplementedError("YvFp8SwiGLU is an inference forward; call .eval()")
        return yvf.fp8_swiglu(x.contiguous(), *self.packed())
