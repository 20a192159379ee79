"""Sizes past 32 bits: the library takes 32-bit counts, so the calls have to refuse what would wrap around to a smaller one."""
import pytest
import torch

from pisceslx_amd import functional as yvf
from pisceslx_amd import quant

FAR = (1 << 32) + 5


def empty(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def weight(o, i):
    groups = -(-i // 128)
    return quant.PackedFp8Linear(i, o, empty(-(-o // 16), groups, 2048, dtype=torch.uint8),
                                 empty(-(-o // 128), groups, dtype=torch.float32))


@pytest.mark.parametrize("call", [
    lambda: yvf.quantize_fp8_rows(empty(FAR, 1)),
    lambda: yvf.quantize_fp8_rows(empty(FAR // 5, 5, 1)),
    lambda: yvf.fp8_linear(empty(FAR, 1), weight(1, 1)),
    lambda: yvf.fp8_linear(quant.Fp8Rows(1, empty(FAR, 128, dtype=torch.float8_e4m3fn),
                                         empty(1, FAR, dtype=torch.float32)), weight(1, 1)),
    lambda: yvf.fp8_swiglu(empty(FAR, 1), weight(1, 1), weight(1, 1), weight(1, 1)),
    lambda: yvf.swiglu(empty(FAR, 1), empty(2, 1), empty(2, 1), empty(1, 2)),
])
def test_rows(call):
    with pytest.raises(ValueError, match="rows.*2\\^24"):
        call()


@pytest.mark.parametrize("call", [
    lambda: yvf.quantize_fp8_rows(empty(1, FAR)),
    lambda: yvf.fp8_linear(empty(1, FAR), weight(1, FAR)),
    lambda: yvf.fp8_linear(empty(1, 1), weight(FAR, 1)),
    lambda: yvf.fp8_swiglu(empty(1, FAR), weight(1, FAR), weight(1, FAR), weight(FAR, 1)),
    lambda: yvf.fp8_swiglu(empty(1, 1), weight(FAR, 1), weight(FAR, 1), weight(1, FAR)),
    lambda: yvf.swiglu(empty(1, FAR), empty(2, FAR), empty(2, FAR), empty(FAR, 2)),
    lambda: yvf.swiglu(empty(1, 2), empty(FAR, 2), empty(FAR, 2), empty(2, FAR)),
])
def test_features(call):
    with pytest.raises(ValueError, match="features.*2\\^20"):
        call()
