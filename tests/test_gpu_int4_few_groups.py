"""int4_linear with fewer groups of 128 columns than a work-group has wavefronts, and several rounds of outputs."""
import pytest
import torch

from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import pack_linear
from test_gpu_int4_linear import check, randn

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("rows,K,O,dtype", [
    (1, 128, 20000, BF16), (1, 512, 24000, BF16), (16, 896, 4112, F32), (1, 7, 20000, BF16), (2, 3, 30000, F32),
    (4, 300, 8200, BF16), (3, 640, 24560, F32),
])
def test_rounds_of_outputs(cuda, rows, K, O, dtype):
    print(f"int4_linear {dtype} {rows} x {K} x {O}", flush=True)
    pk = pack_linear(randn(1, O, K, dtype=F32) * K ** -0.5)
    x, bias = randn(2, rows, K, dtype=dtype), randn(3, O, dtype=dtype)
    check(x, pk, bias, yvf.int4_linear(x, pk, bias), "rounds")
