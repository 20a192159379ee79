"""int4_linear on numbers near the ends of their type's range."""
import pytest
import torch

from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import pack_linear
from test_gpu_int4_linear import check, randn

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,K,O", [(1, 640, 300), (16, 5001, 700), (48, 777, 300), (300, 1300, 4400), (1100, 4224, 4400),
                                      (2047, 4111, 4100)])  # the last with folded corrections
def test_large_rows(cuda, dtype, rows, K, O):
    """Rows of one sign at 2^120: their sums over a group of columns, 2^127, are numbers still, eight times as
    much is not. Every form gives the outputs that the others give, scaled by a power of two."""
    print(f"int4_linear {dtype} {rows} x {K} x {O} large", flush=True)
    pk = pack_linear(randn(1, O, K, dtype=F32) / K)
    x = (1.0 + randn(2, rows, K, dtype=F32).abs().clamp(max=0.99)).to(dtype)
    y = yvf.int4_linear(x, pk)
    check(x, pk, None, y, "at one")
    big = yvf.int4_linear(x * 2.0 ** 120, pk)
    assert bool(torch.isfinite(big).all())
    assert torch.equal(big * 2.0 ** -120, y)


@pytest.mark.parametrize("rows,K,O", [(2047, 4111, 4100), (4090, 300, 2100), (1921, 8200, 4400), (2048, 4096, 4096)])
def test_folded_corrections(cuda, rows, K, O):
    """Outputs for every CU in 128 x 256 tiles: the corrections of 32 groups at a time, whole and in part."""
    print(f"int4_linear {rows} x {K} x {O} folded", flush=True)
    pk = pack_linear(randn(11, O, K, dtype=F32) * K ** -0.5)
    x, bias = randn(12, rows, K) + 0.5, randn(13, O)
    check(x, pk, bias, yvf.int4_linear(x, pk, bias), "folded")
