"""MI355X-native (gfx950) inference forward of the Yv MoE layer.

Host side: PyTorch modules that mirror the reference interfaces (YvStableMoEGate, YvMoEGate,
YvDynamicMoELayer, YvDeepSeekMoELayer, YvRMSNorm, the MoE half of YvHybridBlock, linear layers on
4-bit and 8-bit weights, and the dense gated feed-forward block, which has gradients). Native side: libyvmoe.so, hand-written HIP kernels behind the C ABI in include/yvmoe.h.
"""
from . import _lib
from .ffn import YvFp8SwiGLU, YvSwiGLU
from .gate import YvMoEGate, YvStableMoEGate
from .layer import YvDeepSeekMoELayer, YvDynamicMoELayer
from .linear import YvFp8Linear, YvInt4Linear
from .norms import YvHybridBlockMLP, YvRMSNorm
from .quant import (Fp8Rows, PackedExperts, PackedFp8Linear, PackedLinear, pack_experts, pack_fp8_linear, pack_linear,
                    pack_router)

__all__ = ["YvStableMoEGate", "YvMoEGate", "YvDynamicMoELayer", "YvDeepSeekMoELayer",
           "YvRMSNorm", "YvHybridBlockMLP", "YvInt4Linear", "YvFp8Linear", "YvSwiGLU", "YvFp8SwiGLU", "PackedExperts",
           "PackedLinear", "PackedFp8Linear", "Fp8Rows", "pack_experts", "pack_linear", "pack_fp8_linear",
           "pack_router", "_lib"]
