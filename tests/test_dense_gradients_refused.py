"""What would lose a gradient without a word is refused: on the host, before anything is computed."""
import pytest
import torch
from torch.autograd import forward_ad

from pisceslx_amd import YvFp8SwiGLU, YvHybridBlockMLP, YvSwiGLU
from pisceslx_amd import functional as yvf
from pisceslx_amd import norms, quant


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


def operands(N=3, K=72, O=40):
    """Of 8-bit calls: each a list of its tensors and the call on them."""
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    matrix = lambda o, i: torch.ones(-(-o // 128), -(-i // 128))
    weight = lambda o, i, s: quant.PackedFp8Linear(i, o, torch.zeros(-(-o // 16), -(-i // 128), 2048, dtype=torch.uint8), s)
    return {
        "rows": ([bf(N, K)], yvf.quantize_fp8_rows),
        "linear": ([bf(N, K), matrix(O, K), bf(O), bf(N, O)],
                   lambda x, s, b, out: yvf.fp8_linear(x, weight(O, K, s), b, out)),
        "linear of rows": ([torch.ones(1, N), matrix(O, K), bf(O), bf(N, O)],
                           lambda xs, s, b, out: yvf.fp8_linear(
                               quant.Fp8Rows(K, torch.zeros(N, 128, dtype=torch.float8_e4m3fn), xs), weight(O, K, s), b, out)),
        "block": ([bf(N, K), matrix(O, K), matrix(O, K), matrix(K, O), bf(N, K)],
                  lambda x, g, u, d, out: yvf.fp8_swiglu(x, weight(O, K, g), weight(O, K, u), weight(K, O, d), out)),
    }


@pytest.mark.parametrize("name,which", [(n, i) for n, (ts, _) in operands().items() for i in range(len(ts))])
def test_gradients_of_8_bit_operands(name, which):
    """A gradient of any operand is refused, not only of x; without gradients the next check speaks."""
    ts, call = operands()[name]
    ts[which].requires_grad_(True)
    with pytest.raises(NotImplementedError, match="gradient"):
        call(*ts)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU only"):
        call(*ts)


def block_operands(N=3, H=4, F=8):
    return [torch.zeros(N, H), torch.zeros(F, H), torch.zeros(F, H), torch.zeros(H, F)]


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", range(4))
def test_forward_derivatives_of_the_block(which, grad):
    """A tangent of any operand is refused, whether or not one requires a gradient or gradients are on at all."""
    ts = block_operands()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(ValueError, match="GPU only"):
            yvf.swiglu(*ts)
        ts[which] = forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            yvf.swiglu(*ts)


@pytest.mark.parametrize("name,which", [("rows", 0), ("linear", 0), ("linear", 1), ("linear", 2), ("linear of rows", 0),
                                        ("block", 0), ("block", 3)])
def test_forward_derivatives_of_8_bit_operands(name, which):
    ts, call = operands()[name]
    with torch.no_grad(), forward_ad.dual_level():
        ts[which] = forward_ad.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*ts)
