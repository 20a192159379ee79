"""8-bit rows, linear layer and gated block in 64 bits on the CPU, with what a computed result may be off by."""
import torch

GROUP = 128
# The matrix unit's sum of 128 products: off by at most 8.7e-5 of the sum of their sizes over codes of all
# exponents (16 x 16 sums of random bytes measured); 2^-13 is allowed.
UNIT = 2.0 ** -13


def rows(x):
    """(codes float8 [N][groups * 128], scales [groups][N]) by the definition, in fp32 arithmetic."""
    n, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % GROUP)).view(n, -1, GROUP)
    top = v.abs().amax(dim=2)
    s = (top / torch.full_like(top, 448.0)).clamp(min=1e-12)
    return (v / s[:, :, None]).to(torch.float8_e4m3fn).view(n, -1), s.t().contiguous()


def values(codes, scales, features):
    return (codes.float().double() * scales.t().double().repeat_interleave(GROUP, 1))[:, :features]


def weight(codes, scales):
    """64-bit values of a weight's codes [out][in] (bytes) and block scales."""
    o, i = codes.shape
    s = scales.double().repeat_interleave(GROUP, 0)[:o].repeat_interleave(GROUP, 1)[:, :i]
    return codes.view(torch.float8_e4m3fn).double() * s


def product(v, w):
    """(v wᵀ, what the kernels' may be off by before the output's rounding)."""
    return v @ w.t(), UNIT * (v.abs() @ w.abs().t())


def quantized(h, off):
    """64-bit rows h, known to within off, in 8 bits: (values, what the values of h ± off may differ by)."""
    n, f = h.shape
    pad = (0, -f % GROUP)
    v = torch.nn.functional.pad(h, pad).view(n, -1, GROUP)
    d = torch.nn.functional.pad(off, pad).view(n, -1, GROUP)
    top = v.abs().amax(dim=2, keepdim=True)
    s = (top.float() / 448.0).double().clamp(min=1e-12)
    ds = (d.amax(dim=2, keepdim=True) / top.clamp(min=1e-12)) + 2.0 ** -22  # the scale's relative error
    q = (v / s).float().to(torch.float8_e4m3fn).double()
    dv = d / s + (v / s).abs() * ds
    lo = (v / s - dv).clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
    hi = (v / s + dv).clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
    flip = torch.maximum((lo - q).abs(), (hi - q).abs()) + q.abs() * ds
    return (q * s).view(n, -1)[:, :f], (flip * s).view(n, -1)[:, :f]


def block(x, gate, up, down):
    """(y, allowance) of the gated block on 64-bit weights."""
    v = values(*rows(x), x.shape[1])
    (g, dg), (u, du) = product(v, gate), product(v, up)
    s = 1 / (1 + torch.exp(-g))
    h = g * s * u
    # the activation's slope is below 1.1, and exp, its sum and quotient are within eight half steps
    dh = 1.1 * dg * (u.abs() + du) + (g * s).abs() * du + 8 * 2.0 ** -24 * h.abs()
    hv, dhv = quantized(h, dh)
    y, dy = product(hv, down)
    return y, dy + dhv @ down.abs().t()
