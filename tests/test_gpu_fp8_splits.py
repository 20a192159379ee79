"""8-bit products whose contraction is split over work-groups, in the few-row form and in tiles, and the blocks whose g and
u are: sums of the splits with and without a bias, for odd widths, of rows and of Fp8Rows. Tolerances as in
test_gpu_fp8.py."""
import pytest
import torch

import fp8_reference as ref
from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf
from test_gpu_fp8 import check_linear, make_rows, make_weight, packed

pytestmark = pytest.mark.gpu


def up(v, to):
    return -(-v // to) * to


def splits_of_gate_and_up(n, H, F):
    """From the workspace: besides the rows of x and of h as codes and the down product's, it holds h in fp32, or two sums
    of its size a split."""
    l = _lib.lib()
    rest = (l.yvmoe_fp8_swiglu_workspace_bytes(n, H, F) - l.yvmoe_fp8_linear_workspace_bytes(n, F, H)
            - up(n * up(H, 128), 256) - up(n * up(H, 128) // 32, 256))
    planes = rest // (n * up(F, 128) * 4)
    return planes // 2 if planes > 1 else planes  # 0: h goes on as codes


# few rows with 2 and 4 splits, tiles with 8 and 7
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,i,o", [(5, 8200, 301), (48, 16384, 1001), (100, 4096, 301), (333, 4100, 129)])
def test_linear(cuda, n, i, o, bias):
    assert _lib.lib().yvmoe_fp8_linear_rows_workspace_bytes(n, i, o) > 0, "a product with splits"
    x, w = make_rows(n, i, n + i), make_weight(o, i, o)
    b = torch.randn(o, generator=torch.Generator().manual_seed(o)).to(torch.bfloat16) if bias else None
    p, bc, buf = packed(w, cuda), None if b is None else b.to(cuda), torch.full((n + 2, o), 7.0, dtype=torch.bfloat16, device=cuda)
    got = yvf.fp8_linear(x.to(cuda), p, bc, out=buf[:n])
    assert (buf[n:] == 7).all()
    check_linear(got, x, w, b, f"linear {n} x {i} x {o}")
    rows = yvf.quantize_fp8_rows(x.to(cuda))
    for _ in range(3):
        assert torch.equal(yvf.fp8_linear(rows, p, bc), got)


# few rows: codes of h in a launch of their own; tiles: on the bf16 unit (few h) and on the 8-bit one
@pytest.mark.parametrize("n,H,F", [(48, 2048, 300), (100, 2048, 300), (300, 4096, 1100)])
def test_block(cuda, n, H, F):
    assert splits_of_gate_and_up(n, H, F) > 1
    block(cuda, n, H, F)


def test_block_of_few_values(cuda):
    """One code of h on the other side of a border is 0.006 of y here: g and u have to be fp32's."""
    assert splits_of_gate_and_up(111, 768, 32) == 1
    block(cuda, 111, 768, 32)


def block(cuda, n, H, F):
    x, ws = make_rows(n, H, n + H + F), [make_weight(F, H, 1), make_weight(F, H, 2), make_weight(H, F, 3)]
    p = [packed(w, cuda) for w in ws]
    got = yvf.fp8_swiglu(x.to(cuda), *p)
    y, off = ref.block(x, *(ref.weight(*w) for w in ws))
    d = (got.double().cpu() - y).abs()
    worst = float((d / (2.0 ** -8 * (y.abs() + off) + off + 1e-30)).max())
    rel = float(d.norm() / y.norm())
    print(f"block {n} x {H} x {F}: worst / bound {worst:.3f}, rel {rel:.2e}", flush=True)
    assert torch.isfinite(got).all() and worst <= 1 and rel <= 3.2e-3
    for _ in range(3):
        assert torch.equal(yvf.fp8_swiglu(x.to(cuda), *p), got)


@pytest.mark.parametrize("n,i,o", [(48, 16384, 1001), (100, 4096, 301)])
def test_rows_that_are_no_numbers(cuda, n, i, o):
    x, p = make_rows(n, i, 4), packed(make_weight(o, i, 5), cuda)
    clean = yvf.fp8_linear(x.to(cuda), p)
    x[1, i - 1] = float("nan")
    x[2, 130] = -float("inf")
    got = yvf.fp8_linear(x.to(cuda), p).cpu()
    keep = torch.ones(n, dtype=torch.bool)
    keep[1:3] = False
    assert torch.equal(got[keep], clean.cpu()[keep]) and torch.isnan(got[1:3]).all()
