"""The activation and its derivative at gates far below zero.

g is an input times 1, so exact, u is 1 and the down weight 1. For g from -87.3 up the sigmoid s is a normal number within
six half steps: silu within 7 x 2^-24 and the derivative s + g s (1 - s) within 10 x 2^-24 relative (s's own, the product,
the sum, whose terms are at most 1.02 of it here, and the last product). The block's products may flush terms of an
operand below 2^-126: 2^-125 is allowed. Below -87.3 s is less than the smallest normal number, 2^-126, and may be off by
as much, times |g| <= 89; below -89 both results are 0 by all means: |g| exp(g) is under 2e-37."""
import pytest
import torch

from pisceslx_amd import functional as yvf
from pisceslx_amd import quant

pytestmark = pytest.mark.gpu

FAR = [-87.0, -87.5, -88.0, -88.5, -88.7, -88.8, -89.0, -95.0, -103.0, -104.0, -104.5, -110.0, -1e3, -1e4, -1e20, -1e30, -1e35,
       -3e38]


def gates(n):
    return torch.cat([torch.linspace(-87.2, -60, n - len(FAR)), torch.tensor(FAR)])


def allowed(g, want, half_steps):
    near = g >= -87.3
    return torch.where(near, half_steps * 2.0 ** -24 * want.abs(), torch.where(g >= -89, 90 * 2.0 ** -126, 2e-37)) + 2.0 ** -125


# few rows, operands as they lie (hidden and ffn multiples of 4), packed ones
@pytest.mark.parametrize("n,H,F", [(30, 2, 1), (30, 4, 4), (64, 4, 4), (4000, 4, 4), (4000, 2, 1)])
def test_fp32(cuda, n, H, F):
    g = gates(n)
    x = torch.zeros(n, H)
    x[:, 0], x[:, 1] = g, 1
    wg, wu, wd = torch.zeros(F, H), torch.zeros(F, H), torch.zeros(H, F)
    wg[0, 0] = wu[0, 1] = wd[0, 0] = 1
    dy = torch.zeros(n, H)
    dy[:, 0] = 1
    leaves = [t.to(cuda).requires_grad_(True) for t in (x, wg, wu, wd)]
    y = yvf.swiglu(*leaves)
    dx, = torch.autograd.grad(y, leaves[:1], dy.to(cuda))
    d = g.double()
    s = 1 / (1 + torch.exp(-d))
    for name, got, want, half in (("silu", y[:, 0], d * s, 7), ("derivative", dx[:, 0], s * (1 + d * (1 - s)), 10),
                                  ("du", dx[:, 1], d * s, 7)):
        off = (got.detach().cpu().double() - want).abs()
        worst = (off / allowed(d, want, half)).max()
        print(f"{name} of {n} rows, {H} x {F}: worst / bound {float(worst):.3f}", flush=True)
        assert float(worst) <= 1, (name, [(float(a), float(b)) for a, b in zip(g[-len(FAR):], got[-len(FAR):])])


@pytest.mark.parametrize("n", [30, 300])
def test_bf16(cuda, n):
    """h and y are each rounded once, 2^-8 at most."""
    g = gates(n).to(torch.bfloat16)
    x = torch.stack([g, torch.ones(n, dtype=torch.bfloat16)], 1)
    args = [t.to(torch.bfloat16).to(cuda) for t in (x, torch.tensor([[1.0, 0.0]]), torch.tensor([[0.0, 1.0]]),
                                                    torch.tensor([[1.0], [0.0]]))]
    y = yvf.swiglu(*args)[:, 0].cpu().double()
    d = g.double()
    want = d / (1 + torch.exp(-d))
    off = (y - want).abs()
    assert bool((off <= allowed(d, want, 7) * (1 + 2.0 ** -7) + 2.1 * 2.0 ** -8 * want.abs()).all())


@pytest.mark.parametrize("n", [4, 70])
@pytest.mark.parametrize("g", [-100.0, -1e4, -1e30, -3e38])
def test_8_bits(cuda, n, g):
    """h is far below the smallest scale's smallest code (1e-12 x 2^-9): y is 0."""
    H = F = 128
    one = torch.zeros(F, H)
    one[:, 0] = 1
    q = lambda v, s: quant.pack_fp8_linear_codes((v * 448).to(torch.float8_e4m3fn), torch.tensor([[s / 448]]), v.shape[1]).to(cuda)
    x = torch.zeros(n, H, dtype=torch.bfloat16)
    x[:, 0] = 1
    y = yvf.fp8_swiglu(x.to(cuda), q(-one, -g), q(one, 1.0), q(torch.eye(H, F), 1.0))
    assert not y.any(), float(y.abs().max())
