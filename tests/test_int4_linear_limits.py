"""int4_linear's limits as Python callers meet them."""
import pytest
import torch

from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import pack_linear


@pytest.mark.parametrize("rows", [(1 << 30) + 1, 1 << 32, (1 << 32) + 5])
def test_rows_past_the_limit(rows):
    """More rows than a call takes are refused, not cut to 32 bits (5 of 2^32 + 5 would be computed)."""
    x = torch.zeros(1, 1, dtype=torch.bfloat16).expand(rows, 1)
    with pytest.raises(ValueError, match="rows"):
        yvf.int4_linear(x, pack_linear(torch.ones(1, 1)))
