"""int4_linear's limits as Python callers meet them."""
import pytest
import torch

from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import PackedLinear, pack_linear


@pytest.mark.parametrize("rows", [(1 << 30) + 1, 1 << 32, (1 << 32) + 5])
def test_rows_past_the_limit(rows):
    """More rows than a call takes are refused, not cut to 32 bits (5 of 2^32 + 5 would be computed)."""
    x = torch.zeros(1, 1, dtype=torch.bfloat16).expand(rows, 1)
    with pytest.raises(ValueError, match="rows"):
        yvf.int4_linear(x, pack_linear(torch.ones(1, 1)))


@pytest.mark.parametrize("change", [
    dict(codes=lambda t: t[:1]), dict(codes=lambda t: t[:, :1]), dict(codes=lambda t: t[..., :512]),
    dict(codes=lambda t: t.view(torch.int8)), dict(scales=lambda t: t[:1]), dict(scales=lambda t: t[..., :8]),
    dict(scales=lambda t: t.float()), dict(in_features=lambda n: n + 128), dict(out_features=lambda n: n + 16),
    dict(in_features=lambda n: 0), dict(out_features=lambda n: 0),
])
def test_a_weight_that_does_not_fit_its_sizes(change):
    """Tensors smaller than the sizes say would be read past their ends."""
    pk = pack_linear(torch.ones(30, 200))
    fields = dict(in_features=pk.in_features, out_features=pk.out_features, codes=pk.codes, scales=pk.scales)
    PackedLinear(**fields)
    for name, f in change.items():
        fields[name] = f(fields[name])
    with pytest.raises(ValueError):
        PackedLinear(**fields)
