"""MI355X-native (gfx950) inference forward of the Yv MoE layer.

Host side: PyTorch modules that mirror the reference interfaces (YvStableMoEGate, YvMoEGate,
YvDynamicMoELayer, YvDeepSeekMoELayer, YvRMSNorm, the MoE half of YvHybridBlock, and a linear layer
on 4-bit weights). Native side: libyvmoe.so, hand-written HIP kernels behind the C ABI in include/yvmoe.h.
"""
from . import _lib
from .gate import YvMoEGate, YvStableMoEGate
from .layer import YvDeepSeekMoELayer, YvDynamicMoELayer
from .linear import YvInt4Linear
from .norms import YvHybridBlockMLP, YvRMSNorm
from .quant import PackedExperts, PackedLinear, pack_experts, pack_linear, pack_router

__all__ = ["YvStableMoEGate", "YvMoEGate", "YvDynamicMoELayer", "YvDeepSeekMoELayer",
           "YvRMSNorm", "YvHybridBlockMLP", "YvInt4Linear", "PackedExperts", "PackedLinear", "pack_experts",
           "pack_linear", "pack_router", "_lib"]
