"""Blocks and biases that the layers on packed weights have no place for are refused when they are loaded, on the CPU."""
import pytest
import torch
import torch.nn as nn

from pisceslx_amd import YvFp8Linear, YvFp8SwiGLU, YvInt4Linear, YvSwiGLU


def block(gate=(64, 96), up=(64, 96), down=(96, 64), biased=()):
    m = nn.Module()
    for n, size in (("gate_proj", gate), ("up_proj", up), ("down_proj", down)):
        setattr(m, n, nn.Linear(*size, bias=n in biased))
    return m


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
def test_biases(name):
    """A bias would be left out of the results."""
    with pytest.raises(ValueError, match=f"{name} has a bias"):
        YvFp8SwiGLU.from_block(block(biased=(name,)))


@pytest.mark.parametrize("sizes", [dict(up=(64, 97)), dict(up=(65, 96)), dict(down=(97, 64)), dict(down=(96, 65))])
def test_sizes(sizes):
    with pytest.raises(ValueError, match="no gated block"):
        YvFp8SwiGLU.from_block(block(**sizes))


def test_what_has_a_place():
    for m in (block(), YvSwiGLU(64, 96)):
        packed = YvFp8SwiGLU.from_block(m)
        assert (packed.hidden_size, packed.intermediate_size) == (64, 96)
        assert not packed.training and all(p.bias is None for p in packed.children())


@pytest.mark.parametrize("layer", [YvFp8Linear, YvInt4Linear])
@pytest.mark.parametrize("shape", [(1,), (), (39,), (1, 40)])
def test_bias_of_another_shape(shape, layer):
    """A checkpoint's bias is the layer's or refused: one value is not spread over all outputs, and nothing is loaded."""
    m = layer(64, 40)
    codes = m.codes.clone()
    with pytest.raises(ValueError, match="p.bias"):
        m.load_reference_state_dict({"p.weight": torch.ones(40, 64), "p.bias": torch.ones(shape)}, "p")
    assert torch.equal(m.codes, codes) and int(m.bias.count_nonzero()) == 0
