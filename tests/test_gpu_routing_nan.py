"""Tokens whose logits are not numbers: their choices are experts, as the oracle has them, and nothing is written
outside the routing."""
import numpy as np
import pytest
import torch

from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf
from test_gpu_few import make_experts, make_router, randn
from test_gpu_few_module import make_layer
from test_gpu_routing import _router

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def logits_with_bad_rows(N, E, seed):
    z = (np.random.default_rng(seed).standard_normal((N, E)) * 1.7).astype(np.float32)
    z[0] = NAN
    z[N // 2] = -INF
    z[N // 3, E // 2] = INF
    z[N - 1, : E // 2] = NAN  # the other experts are candidates
    return z


@pytest.mark.parametrize("N,E,k", [(12, 8, 2), (100, 64, 6), (256, 200, 12), (300, 64, 6), (2000, 256, 16)])
@pytest.mark.parametrize("cap", [-1, 3])
def test_route(cuda, oracle, N, E, k, cap):
    print(f"route with NaN N={N} E={E} k={k} cap={cap}", flush=True)
    z = logits_with_bad_rows(N, E, N + E)
    g = yvf.route(torch.from_numpy(z).cuda(), _router(E, k, cap < 0), predictor=False, capacity_override=cap)
    torch.cuda.synchronize()
    o = oracle.route(z, k, cap)
    assert np.array_equal(g.indices.cpu().numpy(), o.indices.astype(np.int64))
    for name in ("counts", "offsets", "perm", "pos"):
        assert np.array_equal(getattr(g, name).cpu().numpy(), getattr(o, name)), name
    w = g.weights.cpu().numpy()
    if cap < 0:
        assert np.array_equal(np.isnan(w), np.isnan(o.weights))
        assert np.array_equal(w[~np.isnan(w)], o.weights[~np.isnan(w)])
    bad = [0, N // 2, N // 3]
    assert np.isnan(w[bad]).all() and not np.isnan(np.delete(w, bad, axis=0)).any()


@pytest.mark.parametrize("fixed", [True, False])
@pytest.mark.parametrize("fmt", ["f32", "bf16", "int8", "int4", "fp8"])
@pytest.mark.parametrize("S", [0, 1])
def test_few_tokens(cuda, fmt, fixed, S):
    """NaN and infinity in a token: no numbers in its outputs, and the routing of the general form. Without a
    capacity the others keep their bits."""
    N, H, E, k = 9, 512, 24, 3
    dt = torch.float32 if fmt == "f32" else torch.bfloat16
    ex = make_experts(fmt, E, S, H, 256, 61)
    st, _ = make_router(E, H, k, dt, 62, fixed=fixed, min_capacity=1)
    mix, x = torch.ones(S, device="cuda") if S else None, randn(63, N, H, dtype=dt)
    want = yvf.moe_forward_few(x, st, ex, mix, None)
    x[2], x[5, 100], x[7] = NAN, INF, -INF
    out, shared, rt = yvf.moe_forward_few(x, st, ex, mix, None)
    general = yvf.moe_forward(x, st, ex, mix, None)
    keep = [i for i in range(N) if i not in (2, 5, 7)]
    assert bool(torch.isnan(out[[2, 5, 7]]).all()) and bool(torch.isfinite(out[keep]).all())
    assert bool(torch.isnan(general[0][[2, 5, 7]]).all()) and bool(torch.isfinite(general[0][keep]).all())
    if S:
        assert bool(torch.isnan(shared[2]).all()) and bool(torch.isfinite(shared[keep]).all())
    for name in ("indices", "counts", "offsets", "perm", "pos", "capacity"):
        assert torch.equal(getattr(rt, name), getattr(general[2], name)), name
    assert bool((rt.indices >= 0).all()) and bool((rt.indices < E).all())
    assert bool(torch.isnan(rt.weights[[2, 5, 7]]).all())
    if fixed:
        assert torch.equal(out[keep], want[0][keep])
        assert torch.equal(rt.weights[keep], want[2].weights[keep])


@pytest.mark.parametrize("router", ["stable", "moegate"])
@pytest.mark.parametrize("few", [0, 16])
@pytest.mark.parametrize("N", [1, 7, 16])
def test_layers(cuda, router, few, N):
    layer = make_layer(router, "int8", few)
    if router == "moegate":
        layer.router._path_moe_stage_size = 1
    x = randn(71, 1, N, layer.hidden_size)
    x[0, N - 1] = NAN
    out, _ = layer(x)
    assert bool(torch.isnan(out[0, N - 1]).all()) and bool(torch.isfinite(out[0, :N - 1]).all())
    idx = layer.last_routing.indices
    assert bool((idx >= 0).all()) and bool((idx < layer.num_experts).all())
