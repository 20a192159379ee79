"""The few-token layer keeps 16 bits of h: outputs against 64 bits within a tolerance that one bf16 term, or a
second one in the wrong place, exceeds (tests/test_few_h_model.py)."""
import pytest
import torch

from few_h_reference import dense, exact, excess, rounding_ratio
from pisceslx_amd import functional as yvf
from test_gpu_few import make_experts, make_router, randn, separated

pytestmark = pytest.mark.gpu
FORMATS = ["bf16", "int8", "int4", "fp8"]


def check(got, ref, tol, what):
    a, b = excess(got, ref, tol), rounding_ratio(got, ref)
    print(f"{what}: {a:.3f} of the tolerance, {b:.4f} of the outputs' rounding", flush=True)
    assert a <= 1.0 and b <= 1.1, what


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N,H,E,F,k,S", [
    (1, 256, 8, 256, 2, 1),      # x and h in LDS
    (2, 4096, 6, 256, 2, 0),     # h alone small
    (3, 640, 5, 896, 3, 2),
    (8, 1152, 4, 640, 2, 1),     # full tiles
    (9, 384, 2, 768, 2, 0),      # a tile and one row more
    (16, 256, 3, 1280, 2, 2),    # x in LDS, h past it
    (16, 4096, 12, 384, 3, 1),   # neither
    (13, 2048, 40, 768, 5, 0),
])
def test_experts(cuda, fmt, N, H, E, F, k, S):
    print(f"h terms {fmt} {N} {H} {E} {F} {k} {S}", flush=True)
    ex = make_experts(fmt, E, S, H, F, 1)
    x, skip = randn(2, N, H), randn(3, N, H) if S else None
    g = torch.Generator(device="cuda").manual_seed(4)
    idx = torch.stack([torch.randperm(E, device="cuda", generator=g)[:k] for _ in range(N)])
    w = torch.softmax(randn(5, N, k, dtype=torch.float32), 1)
    mix = torch.softmax(randn(6, S, dtype=torch.float32), 0) if S else None
    out, shared, _ = yvf.experts_few(x, w, idx, ex, mix, skip)
    ref, sref, tol, stol = exact(x, w, idx, lambda e: dense(ex, e), E, mix, skip)
    check(out, ref, tol, "out")
    if S:
        check(shared, sref, stol, "shared")


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N,H,E,F,k,S", [(1, 1024, 16, 512, 4, 1), (7, 512, 8, 384, 2, 1), (16, 2048, 24, 640, 4, 0)])
def test_layer(cuda, fmt, N, H, E, F, k, S):
    print(f"h terms, layer {fmt} {N} {H} {E} {F} {k} {S}", flush=True)
    ex = make_experts(fmt, E, S, H, F, 11)
    st, gate = make_router(E, H, k, torch.bfloat16, 12)
    x, skip = separated(13, N, gate, st, torch.bfloat16), randn(14, N, H) if S else None
    mix = torch.ones(1, device="cuda") if S else None
    out, shared, rt = yvf.moe_forward_few(x, st, ex, mix, skip)
    ref, sref, tol, stol = exact(x, rt.weights, rt.indices, lambda e: dense(ex, e), E, mix, skip)
    check(out, ref, tol, "out")
    if S:
        check(shared, sref, stol, "shared")
