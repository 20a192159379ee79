"""int4_linear against x Wᵀ + b in 64 bits."""
import ctypes

import pytest
import torch

from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import pack_linear, pack_linear_codes, quantize_int4

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def randn(seed, *shape, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def tolerance(x, pk, ref):
    """Half a step of the output's type, and the 32-bit sums: in a group products of up to 31 |x| and the
    24 |x| taken off again, 2 sqrt(128) half-steps of their sum of magnitudes times the scale; over
    the groups 2 sqrt(n) half-steps of the sum of |x w| and of |y|."""
    u32, half = 2.0 ** -24, 2.0 ** -8 if x.dtype == BF16 else 2.0 ** -24
    K, groups = pk.in_features, pk.codes.shape[1]
    xa = torch.nn.functional.pad(x.double().abs(), (0, groups * 128 - K)).view(-1, groups, 128).sum(-1)
    s = pk.scales.double().abs().permute(0, 2, 1).reshape(-1, groups)[:pk.out_features]
    inside = 2 * 128 ** 0.5 * 55 * u32 * (xa @ s.t())
    over = 2 * groups ** 0.5 * u32 * (x.double().abs() @ pk.dequantize(torch.float64).abs().t())
    return half * 1.01 * ref.abs() + inside + over + 4 * u32 * ref.abs() + 1e-30


def check(x, pk, bias, got, what):
    ref = x.double() @ pk.dequantize(torch.float64).t()
    if bias is not None:
        ref = ref + bias.double()
    assert not torch.isnan(got).any(), what
    bad = float(((got.double() - ref).abs() / tolerance(x, pk, ref)).max())
    print(f"{what}: largest error {bad:.3f} of the tolerance", flush=True)
    assert bad <= 1.0, what


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 2, 5, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("K,O", [(128, 16), (1000, 200), (4096, 64), (2048, 1030)])
def test_rows(cuda, dtype, rows, K, O):
    print(f"int4_linear {dtype} {rows} x {K} x {O}", flush=True)
    pk = pack_linear(randn(1, O, K, dtype=F32) * K ** -0.5)
    x, bias = randn(2, rows, K, dtype=dtype), randn(3, O, dtype=dtype)
    check(x, pk, bias, yvf.int4_linear(x, pk, bias), "with bias")
    y = yvf.int4_linear(x, pk)
    check(x, pk, None, y, "without")
    assert torch.equal(y, yvf.int4_linear(x, pk))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 3, 40, 129])
@pytest.mark.parametrize("K", [1, 7, 31, 33, 127, 129, 383, 1153])
@pytest.mark.parametrize("O", [1, 15, 17, 47])
def test_odd_sizes(cuda, dtype, rows, K, O):
    """Widths that end inside a group, a lane's columns and a block of outputs; rows at any address."""
    print(f"int4_linear {dtype} {rows} x {K} x {O}", flush=True)
    pk = pack_linear(randn(4, O, K, dtype=F32))
    # rows of x start at odd elements; what follows the last one is NaN
    buf = torch.full((rows * K + 70,), float("nan"), dtype=dtype, device="cuda")
    buf[3:3 + rows * K] = randn(5, rows * K, dtype=dtype)
    x = buf[3:3 + rows * K].view(rows, K)
    store = torch.full((rows * O + 40,), 3.0, dtype=dtype, device="cuda")
    out = store[5:5 + rows * O].view(rows, O)
    assert yvf.int4_linear(x, pk, out=out) is out
    check(x, pk, None, out, "odd")
    assert bool((store[:5] == 3.0).all()) and bool((store[5 + rows * O:] == 3.0).all())


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_a_wide_layer(cuda, rows):
    """More columns than a wavefront's first chunks, many blocks of outputs."""
    pk = pack_linear(randn(6, 3000, 9000, dtype=F32) * 0.01)
    x = randn(7, rows, 9000)
    check(x, pk, None, yvf.int4_linear(x, pk), f"{rows} x 9000 x 3000")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,K,O", [
    (1, 2000, 33000), (16, 1024, 25000), (16, 4096, 9000), (3, 1021, 8300),   # rows in LDS, several rounds of outputs
    (16, 5001, 700), (16, 14337, 4100), (9, 9999, 9000), (8, 14400, 2000), (2, 40001, 9000),  # rows that do not fit
    (24, 2050, 9000), (32, 5001, 1000), (48, 1537, 17000), (61, 777, 8500),  # two halves of a step, one past the end
    (50, 1300, 300), (100, 1300, 2100), (100, 640, 4200), (200, 777, 8300),  # tiles of 32, 64 and 128 rows
    (128, 5000, 2100), (300, 4224, 8300), (513, 4111, 4400), (1100, 8200, 4400),  # sums of 32 groups and the rest
])
def test_forms(cuda, dtype, rows, K, O):
    print(f"int4_linear {dtype} {rows} x {K} x {O}", flush=True)
    pk = pack_linear(randn(21, O, K, dtype=F32) * K ** -0.5)
    x, bias = randn(22, rows, K, dtype=dtype) + 0.5, randn(23, O, dtype=dtype)
    y = yvf.int4_linear(x, pk, bias)
    check(x, pk, bias, y, "form")
    # the last row alone, in the form of one row
    check(x[-1:], pk, bias, yvf.int4_linear(x[-1:].contiguous(), pk, bias), "last row alone")


def test_offsets_past_32_bits(cuda):
    """Codes, inputs and outputs of more than 4 GiB: the last block of outputs, the last rows."""
    K, O = 65536, 139264  # 4.25 GiB of codes
    ob, groups = O // 16, K // 128
    from pisceslx_amd.quant import PackedLinear
    pk = PackedLinear(K, O, torch.full((ob, groups, 1024), 0x88, dtype=torch.uint8, device="cuda"),
                      torch.ones(ob, groups, 16, dtype=BF16, device="cuda"))
    tail = pack_linear(randn(8, 16, K, dtype=F32))
    pk.codes[-1], pk.scales[-1] = tail.codes[0], tail.scales[0]
    x = randn(9, 2, K)
    y = yvf.int4_linear(x, pk)
    assert bool((y[:, :-16] == 0).all())
    check(x, tail, None, y[:, -16:].contiguous(), "last block")
    del pk, y
    rows = (1 << 31) // 65536 + 3  # x of more than 2^31 elements
    small = pack_linear(randn(10, 17, K, dtype=F32))
    x = torch.zeros(rows, K, dtype=BF16, device="cuda")
    x[-2:] = randn(11, 2, K)
    y = yvf.int4_linear(x, small)
    assert bool((y[:-2] == 0).all())
    check(x[-2:], small, None, y[-2:], "last rows")


def test_shapes_and_signs(cuda):
    """Leading dimensions, no rows, zero and negative scales, rows of zeros."""
    pk = pack_linear(randn(12, 40, 256, dtype=F32))
    x = randn(13, 2, 3, 5, 256)
    y = yvf.int4_linear(x, pk)
    assert y.shape == (2, 3, 5, 40)
    assert torch.equal(y.view(30, 40), yvf.int4_linear(x.view(30, 256), pk))
    assert yvf.int4_linear(x[:0], pk).shape == (0, 3, 5, 40)
    assert bool((yvf.int4_linear(torch.zeros_like(x), pk) == 0).all())
    q, s = quantize_int4(randn(14, 40, 256, dtype=F32))
    s[3], s[4] = 0.0, -s[4]
    signed = pack_linear_codes(q, s, 256)
    check(x.view(30, 256), signed, None, yvf.int4_linear(x.view(30, 256), signed), "signs")


def test_a_row_of_nan_stays_alone(cuda):
    pk = pack_linear(randn(15, 48, 512, dtype=F32))
    for rows in (6, 40, 200):
        x = randn(16, rows, 512)
        want = yvf.int4_linear(x, pk)
        x[2, 77] = float("nan")
        y = yvf.int4_linear(x, pk)
        keep = [i for i in range(rows) if i != 2]
        assert torch.equal(y[keep], want[keep]) and torch.isnan(y[2]).all()


@pytest.mark.parametrize("rows", [1, 40, 200])
def test_graph_and_stream(cuda, rows):
    """Captured on another stream and replayed with new rows between eager calls."""
    pk = pack_linear(randn(17, 300, 1024, dtype=F32))
    x, bias = randn(18, rows, 1024), randn(19, 300)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        yvf.int4_linear(x, pk, bias)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = yvf.int4_linear(x, pk, bias)
    for rep in range(4):
        x.copy_(randn(30 + rep, rows, 1024))
        g.replay()
        got = y.clone()
        assert torch.equal(got, yvf.int4_linear(x, pk, bias)), rep
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,K,O", [(1, 300, 40), (16, 5001, 700), (48, 777, 300), (300, 1300, 4400), (1100, 4200, 4400)])
def test_rows_that_are_not_numbers(cuda, dtype, rows, K, O):
    """An infinity or NaN makes its row NaN and leaves the others as they are."""
    pk = pack_linear(randn(31, O, K, dtype=F32))
    x = randn(32, rows, K, dtype=dtype)
    y = yvf.int4_linear(x, pk)
    bad = sorted({0, rows // 2, rows - 1})
    for i, v in zip(bad, (float("inf"), float("nan"), float("-inf"))):
        x[i, (i * 37 + 5) % K] = v
    z = yvf.int4_linear(x, pk)
    assert bool(torch.isnan(z[bad]).all())
    good = [i for i in range(rows) if i not in bad]
    assert torch.equal(z[good], y[good])
