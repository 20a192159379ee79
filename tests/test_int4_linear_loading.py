"""Loading a YvInt4Linear from a reference state."""
import pytest
import torch

from pisceslx_amd import YvInt4Linear


def test_a_bias_is_not_dropped():
    """A checkpoint's bias that the layer has no place for is refused, and leaves the layer as it was."""
    w, b = torch.randn(40, 256), torch.randn(40)
    m = YvInt4Linear(256, 40, bias=False)
    before = m.codes.clone()
    with pytest.raises(ValueError, match="p.bias"):
        m.load_reference_state_dict({"p.weight": w, "p.bias": b}, "p")
    assert torch.equal(m.codes, before)
    m.load_reference_state_dict({"p.weight": w}, "p")
    assert not torch.equal(m.codes, before)
    with_bias = YvInt4Linear(256, 40)
    with pytest.raises(KeyError):
        with_bias.load_reference_state_dict({"p.weight": w}, "p")
    assert torch.equal(with_bias.codes, before)
