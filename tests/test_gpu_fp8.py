"""8-bit rows, the 8-bit linear layer and the gated block on 8-bit weights against 64-bit evaluations.

Tolerances. Codes and scales are equal. A linear output is off by the unit's sums (fp8_reference.UNIT of the sum of
the products' sizes), the fp32 sum over the groups (2^-24 a group) and its own rounding, 2^-8 at most, uniform over
half a step: 2^-8 / sqrt(3) = 2.26e-3 rms at the very most. The block's y is off by that and by the codes of h
that lie within the error of g and u from a border (fp8_reference.quantized). In 2-norm such flips are few: g and u
are off by about 2e-5, a code's half step is 2^-5 to 2^-4 of it, so about one code in a thousand flips, by at
most 2^-3 relative (0.07 rms): 0.07 / sqrt(1000) = 2.2e-3, with the output's rounding 3.2e-3.
"""
import math

import pytest
import torch

import fp8_reference as ref
from pisceslx_amd import functional as yvf
from pisceslx_amd import quant

pytestmark = pytest.mark.gpu


def make_rows(n, k, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, k, generator=g) * (0.25 + torch.rand(n, 1, generator=g))
    x[:, 3::41] *= 8
    return x.to(dtype)


def make_weight(o, i, seed):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(o, i, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    s = (0.5 + torch.rand(-(-o // 128), -(-i // 128), generator=g)) * (0.01 / math.sqrt(i))
    return q, s


def packed(w, dev):
    return quant.pack_fp8_linear_codes(w[0], w[1], w[0].shape[1]).to(dev)


def same_codes(got, want):
    """Equal as bytes, a NaN with either sign and any bits."""
    a, b = got.cpu().float(), want.float()
    nan = torch.isnan(b)
    return torch.equal(torch.isnan(a), nan) and torch.equal(got.cpu().view(torch.uint8)[~nan],
                                                            want.view(torch.uint8)[~nan])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 128), (2, 127), (3, 129), (5, 8), (7, 4096), (64, 200), (33, 1000),
                                 (17, 4095), (300, 516), (1, 20000)])
def test_rows(cuda, n, k, dtype):
    x = make_rows(n, k, n + k, dtype)
    got = yvf.quantize_fp8_rows(x.to(cuda))
    q, s = ref.rows(x)
    assert same_codes(got.codes, q)
    assert torch.equal(got.scales.cpu(), s)


def test_rows_values(cuda):
    """Zeros, values below the smallest scale, subnormals, the largest ones, ties, infinities and NaN."""
    x = make_rows(12, 384, 1, torch.float32)
    x[0, :128] = 0
    x[1, 128:256] = 1e-14
    x[2, :128] = 1e-40
    x[3, 256:] = 3e38
    x[4, 5] = math.inf
    x[5, 200] = math.nan
    x[6, 300] = -math.inf
    # halfway between codes: 448, and 17 / 16 of powers of two
    x[7, :128] = torch.arange(128).float().remainder(20).sub(6).exp2() * 17 / 16
    x[7, 0] = 448.0
    x[8, :128] = -x[7, :128]
    x[9] = -0.0
    for t in (x, x.to(torch.bfloat16)):
        got = yvf.quantize_fp8_rows(t.to(cuda))
        q, s = ref.rows(t)
        assert same_codes(got.codes, q)
        assert torch.equal(torch.nan_to_num(got.scales.cpu(), -1.0), torch.nan_to_num(s, -1.0))


def test_rows_of_any_alignment(cuda):
    x = make_rows(9, 264, 3).to(cuda)
    flat = torch.zeros(x.numel() + 1, dtype=x.dtype, device=cuda)
    flat[1:].copy_(x.view(-1))
    a, b = yvf.quantize_fp8_rows(flat[1:].view_as(x)), yvf.quantize_fp8_rows(x)
    assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    c = yvf.quantize_fp8_rows(x.view(3, 3, 264))
    assert torch.equal(c.codes.view(torch.uint8), b.codes.view(torch.uint8))


LINEAR = [(1, 1, 1), (1, 128, 16), (1, 4096, 272), (2, 100, 40), (7, 1000, 301), (15, 384, 128), (16, 2048, 130),
          (17, 256, 144), (31, 129, 17), (33, 640, 200), (48, 1536, 96), (64, 128, 33), (65, 300, 257), (100, 512, 129),
          (129, 1152, 64), (255, 200, 300), (300, 384, 1000)]


def check_linear(got, x, w, bias, name):
    v = ref.values(*ref.rows(x), x.shape[1])
    y, off = ref.product(v, ref.weight(*w))
    if bias is not None:
        y = y + bias.double()
    off = off + 2.0 ** -24 * (w[1].shape[1] + 2) * (off / ref.UNIT + y.abs())
    d = (got.double().cpu() - y).abs()
    worst = float((d / (2.0 ** -8 * (y.abs() + off) + off + 1e-30)).max())
    rel = float(d.norm() / y.norm().clamp(min=1e-300))
    print(f"{name}: worst / bound {worst:.3f}, rel {rel:.2e}", flush=True)
    assert torch.isfinite(got).all() and worst <= 1
    assert rel <= (2.3e-3 if y.numel() > 64 else 2.0 ** -8 * 1.01)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,i,o", LINEAR)
def test_linear(cuda, n, i, o, bias):
    x, w = make_rows(n, i, n + i), make_weight(o, i, o)
    b = torch.randn(o, generator=torch.Generator().manual_seed(o)).to(torch.bfloat16) if bias else None
    p = packed(w, cuda)
    got = yvf.fp8_linear(x.to(cuda), p, None if b is None else b.to(cuda))
    assert got.shape == (n, o) and got.dtype == torch.bfloat16
    check_linear(got, x, w, b, f"linear {n} x {i} x {o}")
    # rows quantized before: the same bits
    again = yvf.fp8_linear(yvf.quantize_fp8_rows(x.to(cuda)), p, None if b is None else b.to(cuda))
    assert torch.equal(again, got)


# tiles of 256, whole and partial
@pytest.mark.parametrize("n,i,o", [(2048, 512, 5120), (2100, 1000, 4999), (5000, 256, 2100)])
def test_linear_large(cuda, n, i, o):
    x, w = make_rows(n, i, n + i), make_weight(o, i, o)
    p = packed(w, cuda)
    got = yvf.fp8_linear(x.to(cuda), p)
    check_linear(got, x, w, None, f"linear {n} x {i} x {o}")
    assert torch.equal(yvf.fp8_linear(x.to(cuda), p), got)


def test_linear_empty_and_leading(cuda):
    w = make_weight(40, 72, 1)
    p = packed(w, cuda)
    assert yvf.fp8_linear(torch.empty(0, 72, dtype=torch.bfloat16, device=cuda), p).shape == (0, 40)
    x = make_rows(6, 72, 2).to(cuda)
    out = torch.empty(2, 3, 40, dtype=torch.bfloat16, device=cuda)
    assert yvf.fp8_linear(x.view(2, 3, 72), p, out=out) is out
    assert torch.equal(out.view(6, 40), yvf.fp8_linear(x, p))


@pytest.mark.parametrize("n", [3, 40, 200])
def test_linear_rows_that_are_no_numbers(cuda, n):
    x, w = make_rows(n, 300, 4), make_weight(72, 300, 5)
    p = packed(w, cuda)
    clean = yvf.fp8_linear(x.to(cuda), p)
    x[1, 299] = math.nan
    x[2, 130] = -math.inf
    got = yvf.fp8_linear(x.to(cuda), p).cpu()
    keep = torch.ones(n, dtype=torch.bool)
    keep[1:3] = False
    assert torch.equal(got[keep], clean.cpu()[keep]) and torch.isnan(got[1:3]).all()


def test_rows_behind_the_last_one_stay(cuda):
    """Outputs end where they end: what lies behind the last row is not written."""
    w = make_weight(24, 128, 6)
    p = packed(w, cuda)
    for n in (3, 20, 70, 130):
        buf = torch.full((n + 5, 24), 7.0, dtype=torch.bfloat16, device=cuda)
        yvf.fp8_linear(make_rows(n, 128, 7).to(cuda), p, out=buf[:n])
        assert (buf[n:] == 7).all()


def test_weights_of_packed_experts(cuda):
    """An expert's fp8 matrices are such weights as they are."""
    g = torch.Generator().manual_seed(8)
    mats = [(torch.randn(256, 384, generator=g), torch.randn(256, 384, generator=g),
             torch.randn(384, 256, generator=g)) for _ in range(2)]
    pk = quant.pack_experts(mats, 2, quant.FORMAT_BY_NAME["fp8"], device=cuda)
    x = make_rows(20, 384, 9).to(cuda)
    ours = [quant.PackedFp8Linear(384, 256, pk.w_gate[1].view(16, 3, 2048), pk.s_gate[1]),
            quant.PackedFp8Linear(384, 256, pk.w_up[1].view(16, 3, 2048), pk.s_up[1]),
            quant.PackedFp8Linear(256, 384, pk.w_down[1].view(24, 2, 2048), pk.s_down[1])]
    plain = [quant.pack_fp8_linear(m.to(cuda)) for m in mats[1]]
    assert torch.equal(yvf.fp8_swiglu(x, *ours), yvf.fp8_swiglu(x, *plain))
    for a, b in zip(ours, plain):
        assert torch.equal(a.dequantize(), b.dequantize())


BLOCKS = [(1, 1, 1), (1, 4096, 1408), (2, 100, 300), (5, 384, 512), (16, 640, 384), (20, 129, 1000), (48, 512, 640),
          (64, 200, 130), (65, 256, 384), (130, 300, 500), (300, 512, 1027), (1100, 256, 5120), (2500, 384, 2600)]


@pytest.mark.parametrize("n,H,F", BLOCKS)
def test_block(cuda, n, H, F):
    x, ws = make_rows(n, H, n + H + F), [make_weight(F, H, 1), make_weight(F, H, 2), make_weight(H, F, 3)]
    p = [packed(w, cuda) for w in ws]
    got = yvf.fp8_swiglu(x.to(cuda), *p)
    y, off = ref.block(x, *(ref.weight(*w) for w in ws))
    d = (got.double().cpu() - y).abs()
    worst = float((d / (2.0 ** -8 * (y.abs() + off) + off + 1e-30)).max())
    rel = float(d.norm() / y.norm())
    print(f"block {n} x {H} x {F}: worst / bound {worst:.3f}, rel {rel:.2e}", flush=True)
    assert torch.isfinite(got).all() and worst <= 1
    assert rel <= (3.2e-3 if y.numel() > 1000 else 2e-2)  # one flipped code counts among few
    assert torch.equal(yvf.fp8_swiglu(x.to(cuda), *p), got)


@pytest.mark.parametrize("n", [4, 100, 2500])
def test_block_rows_that_are_no_numbers(cuda, n):
    x = make_rows(n, 256, 11)
    p = [packed(make_weight(o, i, o + i), cuda) for o, i in ((2600, 256), (2600, 256), (256, 2600))]
    clean = yvf.fp8_swiglu(x.to(cuda), *p)
    x[2, 0] = math.nan
    got = yvf.fp8_swiglu(x.to(cuda), *p).cpu()
    keep = torch.ones(n, dtype=torch.bool)
    keep[2] = False
    assert torch.equal(got[keep], clean.cpu()[keep]) and torch.isnan(got[2]).all()


@pytest.mark.parametrize("n", [1, 40, 200])
def test_captured(cuda, n):
    """A projection, a gated block and a projection in a row, captured and replayed on new rows."""
    H, F = 256, 384
    ps = [packed(make_weight(o, i, o), cuda) for o, i in ((H, H), (F, H), (F, H), (H, F), (136, H))]

    def run(x):
        return yvf.fp8_linear(yvf.fp8_swiglu(yvf.fp8_linear(x, ps[0]), *ps[1:4]), ps[4])
    x = make_rows(n, H, 12).to(cuda)
    run(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(x)
    for k in range(4):
        new = make_rows(n, H, 20 + k).to(cuda)
        x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, run(new))


def test_on_another_stream(cuda):
    p = packed(make_weight(64, 256, 1), cuda)
    x = make_rows(30, 256, 2).to(cuda)
    want = yvf.fp8_linear(x, p)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = yvf.fp8_linear(x, p)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("n,o", [(2090, 4999), (2500, 5132), (130, 4107), (70, 1003)])
def test_ends_of_tiles(cuda, n, o):
    """Outputs of odd widths leave the tiles whole, with a bias, and nothing behind the last row is written."""
    x, w = make_rows(n, 200, n), make_weight(o, 200, o)
    b = torch.randn(o, generator=torch.Generator().manual_seed(o)).to(torch.bfloat16)
    buf = torch.full((n + 3, o), 7.0, dtype=torch.bfloat16, device=cuda)
    p = packed(w, cuda)
    yvf.fp8_linear(x.to(cuda), p, b.to(cuda), out=buf[:n])
    assert (buf[n:] == 7).all()
    check_linear(buf[:n], x, w, b, f"linear {n} x 200 x {o}")


@pytest.mark.parametrize("n", [40, 40000])
def test_rows_by_every_kind_of_scale(cuda, n):
    """Codes are those of the rounded quotient, at scales of all mantissas and beside the borders between codes: each
    group holds 448 s, which makes its scale s, and values at t / 16 s and its fp32 neighbours, t from 16 to 31."""
    g = torch.Generator().manual_seed(n)
    s = torch.randint(0, 1 << 23, (n,), generator=g)
    s[::2] = (s[::2] & ~0xfffff) + torch.randint(-20, 20, (len(s[::2]),), generator=g)  # beside multiples of 1 / 8
    s = (s.clamp(min=0).to(torch.int32) + (127 << 23)).view(torch.float32)
    t = torch.arange(16, 32) / 16.0
    near = (t[None] * s[:, None]).view(torch.int32)[:, :, None] + torch.arange(-3, 4, dtype=torch.int32)
    x = torch.cat([448 * s[:, None], near.view(torch.float32).view(n, -1), torch.zeros(n, 15)], 1)
    x = x * torch.randint(-12, 12, (n, 1), generator=g).float().exp2()
    q, _ = ref.rows(x)
    assert same_codes(yvf.quantize_fp8_rows(x.to(cuda)).codes, q)
