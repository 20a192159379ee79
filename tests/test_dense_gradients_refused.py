"""What would lose a gradient without a word is refused: on the host, before anything is computed."""
import pytest
import torch

from pisceslx_amd import YvFp8SwiGLU, YvHybridBlockMLP, YvSwiGLU
from pisceslx_amd import norms


class Config:
    hidden_size, n_layer = 32, 4


@pytest.mark.parametrize("mlp", [lambda: YvSwiGLU(32, 48), lambda: YvFp8SwiGLU(32, 48)], ids=["block", "fp8"])
def test_half_block_in_training(mlp, monkeypatch):
    """The half block has no gradients: in training mode it raises, whatever its mlp can do by itself."""
    monkeypatch.setattr(norms, "rms_norm_chain", lambda x, *n: x * 1)
    for block in (YvSwiGLU, YvFp8SwiGLU):
        monkeypatch.setattr(block, "forward", lambda self, x: x * 2)
    half = YvHybridBlockMLP(Config, mlp=mlp())
    for h in (half, half.eval().train()):
        with pytest.raises(NotImplementedError, match="YvHybridBlockMLP.*eval"):
            h(torch.zeros(3, 32, requires_grad=True))
    y, loss = half.eval()(torch.ones(3, 32))
    assert y.shape == (3, 32) and float(loss) == 0
    # a mlp that is in eval mode, as those that are packed from a block are, serves in a half block as it is made
    served = YvHybridBlockMLP(Config, mlp=mlp().eval())
    assert torch.equal(served(torch.ones(3, 32))[0], y)
