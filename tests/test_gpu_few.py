"""The few-token layer (moe_forward_few, experts_few) against a plain statement in 64 bits."""
import ctypes

import pytest
import torch

from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import ExpertPacker, FORMAT_BY_NAME, pack_router

pytestmark = pytest.mark.gpu
FORMATS = ["f32", "bf16", "int8", "int4", "fp8"]


def make_experts(fmt, E, S, H, F, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pk = ExpertPacker(FORMAT_BY_NAME[fmt], E, S, H, F, "cuda")
    for e in range(E + S):
        pk.set(e, *[torch.randn(o, i, device="cuda", generator=g) * i ** -0.5
                    for o, i in ((F, H), (F, H), (H, F))])
    return pk.packed


def make_router(E, H, k, dtype, seed, fixed=False, bias=None, dynamic=True, min_capacity=4, factor=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    gate = (torch.randn(E, H, device="cuda", generator=g) * H ** -0.5).to(dtype)
    w1 = torch.randn(64, H, device="cuda", generator=g) * H ** -0.5
    act = _lib.ACT_F32 if dtype == torch.float32 else _lib.ACT_BF16
    b1 = torch.randn(64, device="cuda", generator=g) * 0.1
    w2 = torch.randn(1, 64, device="cuda", generator=g) * 0.1
    st = yvf.RouterState(E, H, k, fixed, dynamic, min_capacity, factor, pack_router(gate, w1, act), b1, w2,
                         torch.zeros(1, device="cuda"), bias)
    return st, gate


def randn(seed, *shape, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def reference(x, w, idx, ex, mix, skip):
    """(out, shared, tolerance of out, of shared) in 64 bits. h is rounded to bf16 for bf16
    activations, as the operator states. Tolerances: half a step of the output's type, and

    * for the sums in 32 bits before h, 2 sqrt(n) half-steps of the sum of |products|, carried on
      through |Wd|;
    * where that moves h over a rounding border, a whole bf16 step (2^-7) of that h: less than one in
      a thousand elements (an error of some 2^-22 against steps of 2^-7), counted as a thousandth of
      the sum of |Wd h| plus four times its largest term."""
    N, H = x.shape
    bf = x.dtype == torch.bfloat16
    u32, half = 2.0 ** -24, 2.0 ** -8 if bf else 2.0 ** -24
    x = x.double()
    out = torch.zeros(N, H, dtype=torch.float64, device="cuda")
    tol, shared, stol = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)

    def expert(e, t, scale, into, tinto):
        g, u, d = ex.dequantize(e, torch.float64)
        xs = x[t]
        gs, us = xs @ g.t(), xs @ u.t()
        err_g = 2 * ex.hidden ** 0.5 * u32 * (xs.abs() @ g.abs().t())
        err_u = 2 * ex.hidden ** 0.5 * u32 * (xs.abs() @ u.abs().t())
        act = torch.nn.functional.silu(gs)
        h = act * us
        err_h = 1.1 * err_g * us.abs() + act.abs() * err_u + 8 * u32 * h.abs()
        if bf:
            h = h.to(torch.bfloat16).double()
        terms = h.abs()
        y = h @ d.t()
        e32 = err_h @ d.abs().t() + 2 * ex.ffn ** 0.5 * u32 * (terms @ d.abs().t())
        if bf:
            big = (terms[:, None, :] * d.abs()[None]).amax(dim=-1)
            e32 = e32 + 2.0 ** -7 * (1e-3 * (terms @ d.abs().t()) + 4 * big)
        s = scale.double()[:, None]
        into.index_add_(0, t, s * y)
        tinto.index_add_(0, t, s.abs() * (e32 + 4 * u32 * y.abs()))

    for e in range(ex.num_routed):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if t.numel():
            expert(e, t, w[t, j], out, tol)
    every = torch.arange(N, device="cuda")
    for s in range(ex.num_shared):
        expert(ex.num_routed + s, every, mix[s].expand(N), shared, stol)
    out, tol = out + shared, tol + stol
    if skip is not None:
        out = out + 0.1 * skip.double()
        tol = tol + 2 * u32 * skip.double().abs()
    return out, shared, tol + half * out.abs() * 1.01 + 4 * u32, stol + half * shared.abs() * 1.01 + 4 * u32


def check(got, want, tol, what):
    assert not torch.isnan(got).any(), what
    bad = (got.double() - want).abs() / tol
    print(f"{what}: largest error {float(bad.max()):.3f} of the tolerance")
    assert float(bad.max()) <= 1.0, what


def separated(seed, N, gate, st, dtype):
    """N tokens none of whose first logits lie closer than 32-bit sums in any order can tell."""
    x = randn(seed, N + 32, st.hidden, dtype=dtype)
    z = x.double() @ gate.double().t()
    if st.bias is not None:
        z = z + st.bias.double()
    z = torch.sort(z, dim=1, descending=True).values[:, :st.top_k + 1]
    if z.shape[1] > 1:
        x = x[(z[:, :-1] - z[:, 1:]).amin(dim=1) > 2e-5]
    return x[:N].contiguous()


def routing_reference(x, gate, st):
    """Indices, weights and capacity by the algorithm, logits in 64 bits."""
    N, E, k = x.shape[0], st.num_experts, st.top_k
    z = x.double() @ gate.double().t()
    if st.bias is not None:
        z = z + st.bias.double()
    p, idx = torch.sort(torch.softmax(z, 1), dim=1, descending=True, stable=True)
    p, idx = p[:, :k], idx[:, :k]
    w = torch.softmax(p, 1)
    return idx, p, w


CASES = [
    # N, H, E, F, k, S
    (1, 256, 8, 256, 2, 1),
    (1, 128, 1, 128, 1, 0),
    (2, 640, 5, 384, 3, 2),
    (5, 1152, 12, 128, 12, 0),
    (7, 384, 100, 640, 7, 1),
    (16, 256, 3, 1280, 2, 8),
    (16, 512, 256, 128, 16, 0),
    (13, 2048, 40, 768, 5, 3),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N,H,E,F,k,S", CASES)
def test_experts_few(cuda, fmt, N, H, E, F, k, S):
    dt = torch.float32 if fmt == "f32" else torch.bfloat16
    ex = make_experts(fmt, E, S, H, F, 1)
    x, skip = randn(2, N, H, dtype=dt), randn(3, N, H, dtype=dt)
    logits = randn(4, N, E, dtype=torch.float32)
    top = torch.topk(logits, k, dim=1)
    w, idx = torch.softmax(top.values, 1).contiguous(), top.indices.contiguous()
    mix = torch.softmax(randn(5, S, dtype=torch.float32), 0) if S else None
    print(f"experts_few {fmt} {N} {H} {E} {F} {k} {S}", flush=True)
    out, shared, invalid = yvf.experts_few(x, w, idx, ex, mix, skip if S else None)
    ref, sref, tol, stol = reference(x, w, idx, ex, mix, skip if S else None)
    check(out, ref, tol, "out")
    assert int(invalid) == 0
    if S:
        check(shared, sref, stol, "shared")
    else:
        assert shared is None
    again = yvf.experts_few(x, w, idx, ex, mix, skip if S else None)[0]
    assert torch.equal(out, again)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "int4", "fp8"])
@pytest.mark.parametrize("H,F", [(64, 64), (192, 320), (1088, 832), (4096, 1408)])
def test_widths(cuda, fmt, H, F):
    """Widths of every remainder of the chunks (multiples of 64, of 128 for int4 and fp8)."""
    if fmt in ("int4", "fp8"):
        H, F = (H + 127) // 128 * 128, (F + 127) // 128 * 128
    N, E, k, S = 3, 6, 2, 1
    ex = make_experts(fmt, E, S, H, F, 11)
    x = randn(12, N, H)
    idx = torch.tensor([[0, 5], [5, 1], [2, 0]], device="cuda")
    w = torch.tensor([[0.7, 0.3], [0.5, 0.5], [1.0, 0.0]], device="cuda").to(torch.bfloat16)
    mix = torch.ones(1, device="cuda")
    print(f"widths {fmt} {H} {F}", flush=True)
    out, shared, _ = yvf.experts_few(x, w, idx, ex, mix)
    ref, sref, tol, stol = reference(x, w.float(), idx, ex, mix, None)
    check(out, ref, tol, "out")
    check(shared, sref, stol, "shared")


@pytest.mark.parametrize("fmt", ["f32", "int4", "int8"])
def test_repeated_and_invalid_indices(cuda, fmt):
    """One expert named by every slot (tiles of 16 rows), indices outside [0, E), zero weights."""
    dt = torch.float32 if fmt == "f32" else torch.bfloat16
    N, H, E, F, k, S = 16, 256, 9, 128, 16, 1
    ex = make_experts(fmt, E, S, H, F, 21)
    x, mix = randn(22, N, H, dtype=dt), torch.ones(1, device="cuda")
    w = torch.rand(N, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(23)) / k
    same = torch.full((N, k), 4, dtype=torch.int64, device="cuda")
    mixed = same.clone()
    mixed[:, 3], mixed[0, 0], mixed[5, 7], mixed[6, :] = -1, E, 1 << 40, -(1 << 40)
    mixed[2, 1:3] = 0
    w[3, :4] = 0.0
    for idx in (same, mixed):
        out, _, invalid = yvf.experts_few(x, w, idx, ex, mix)
        ref, _, tol, _ = reference(x, w, idx, ex, mix, None)
        check(out, ref, tol, f"{fmt} repeated")
        assert int(invalid) == int(((idx < 0) | (idx >= E)).sum())
    out, _, invalid = yvf.experts_few(x, w, torch.full_like(same, -7), ex, mix)
    ref, _, tol, _ = reference(x, w, torch.full_like(same, -7), ex, mix, None)
    check(out, ref, tol, "none valid")
    assert int(invalid) == N * k


LAYERS = [
    # N, H, E, F, k, S, fixed, bias, min_capacity, dynamic
    (1, 1024, 8, 256, 2, 1, False, False, 4, True),
    (16, 512, 8, 128, 2, 1, False, False, 1, True),    # experts past their capacity
    (16, 512, 4, 128, 4, 0, False, False, 2, False),   # every expert past it, static factor
    (16, 512, 4, 128, 2, 0, False, False, 0, False),
    (9, 4096, 64, 128, 6, 2, False, True, 4, True),
    (5, 1920, 200, 128, 12, 0, True, True, 4, True),
    (16, 256, 256, 128, 16, 1, True, False, 4, True),
    (3, 128, 1, 128, 1, 1, False, False, 1, True),
]


@pytest.mark.parametrize("fmt", ["f32", "bf16", "int4"])
@pytest.mark.parametrize("N,H,E,F,k,S,fixed,bias,mincap,dynamic", LAYERS)
def test_layer(cuda, fmt, N, H, E, F, k, S, fixed, bias, mincap, dynamic):
    """Routing as moe_forward's (the same code from the logits on), outputs by the definition."""
    dt = torch.float32 if fmt == "f32" else torch.bfloat16
    ex = make_experts(fmt, E, S, H, F, 31)
    b = randn(32, E, dtype=torch.float32) * 0.5 if bias else None
    st, gate = make_router(E, H, k, dt, 33, fixed, b, dynamic, mincap)
    x, skip = separated(34, N, gate, st, dt), randn(35, N, H, dtype=dt)
    mix = torch.softmax(randn(36, S, dtype=torch.float32), 0) if S else None
    print(f"layer {fmt} {N} {H} {E} {F} {k} {S} {fixed} {bias} {mincap} {dynamic}", flush=True)
    out, shared, rt = yvf.moe_forward_few(x, st, ex, mix, skip if S else None)
    idx, p, w0 = routing_reference(x, gate, st)
    assert torch.equal(rt.indices, idx)
    want = yvf.moe_forward(x, st, ex, mix, skip if S else None)[2]
    for name in ("indices", "counts", "offsets", "perm", "pos", "capacity"):
        assert torch.equal(getattr(rt, name), getattr(want, name)), name
    # weights of probabilities from logits within a few 32-bit steps
    assert (rt.weights - want.weights).abs().max() <= 2.0 ** -18
    if fixed:
        assert (rt.weights.double() - w0).abs().max() <= 2.0 ** -18
    else:
        assert torch.equal(rt.weights == 0, want.weights == 0)
    ref, sref, tol, stol = reference(x, rt.weights, idx, ex, mix, skip if S else None)
    check(out, ref, tol, "out")
    if S:
        check(shared, sref, stol, "shared")


def test_equal_logits_go_to_the_lower_expert(cuda):
    H, E, k = 256, 24, 5
    ex = make_experts("bf16", E, 0, H, 128, 41)
    st, gate = make_router(E, H, k, torch.bfloat16, 42, fixed=True)
    gate[:] = gate[0]
    st.w_router = pack_router(gate, None, _lib.ACT_BF16)
    rt = yvf.moe_forward_few(randn(43, 4, H), st, ex, None, None)[2]
    assert rt.indices.tolist() == [[0, 1, 2, 3, 4]] * 4


def test_no_tokens(cuda):
    ex = make_experts("int8", 6, 1, 128, 128, 51)
    st, _ = make_router(6, 128, 2, torch.bfloat16, 52)
    mix = torch.ones(1, device="cuda")
    out, shared, rt = yvf.moe_forward_few(randn(53, 0, 128), st, ex, mix, None)
    assert out.shape == (0, 128) and shared.shape == (0, 128)
    assert rt.counts.tolist() == [0] * 6 and rt.offsets.tolist() == [0] * 7 and int(rt.capacity) == 4
    out, _, invalid = yvf.experts_few(randn(53, 0, 128), torch.empty(0, 2, device="cuda"),
                                      torch.empty(0, 2, dtype=torch.int64, device="cuda"), ex, mix)
    assert out.shape == (0, 128) and int(invalid) == 0


@pytest.mark.parametrize("fmt", ["bf16", "int8", "fp8"])
def test_a_token_of_nan_stays_alone(cuda, fmt):
    """NaN and infinity in one token leave the others' bits; its own row is NaN."""
    H, E, k, S = 512, 16, 3, 1
    ex = make_experts(fmt, E, S, H, 256, 61)
    st, _ = make_router(E, H, k, torch.bfloat16, 62, fixed=True)
    mix, x = torch.ones(1, device="cuda"), randn(63, 6, H)
    bad = x.clone()
    bad[2] = float("nan")
    good_out = yvf.moe_forward_few(x, st, ex, mix, None)
    out, shared, rt = yvf.moe_forward_few(bad, st, ex, mix, None)
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(rt.indices[keep], good_out[2].indices[keep])
    assert torch.equal(out[keep], good_out[0][keep]) and torch.equal(shared[keep], good_out[1][keep])
    assert torch.isnan(out[2]).all() and torch.isnan(shared[2]).all()


def test_untouched_experts_are_not_read_into_the_result(cuda):
    H, E = 256, 12
    ex = make_experts("int8", E, 0, H, 128, 71)
    x, w = randn(72, 2, H), torch.full((2, 2), 0.5, device="cuda")
    idx = torch.tensor([[3, 7], [7, 3]], device="cuda")
    want = yvf.experts_few(x, w, idx, ex)[0]
    for e in set(range(E)) - {3, 7}:
        for s in (ex.s_gate, ex.s_up, ex.s_down):
            s[e] = float("nan")
    assert torch.equal(yvf.experts_few(x, w, idx, ex)[0], want)


def test_workspace_and_outputs_stay_inside(cuda):
    """Bytes behind the workspace and rows behind the batch keep what they held."""
    H, E, F, k, S, N = 192, 7, 64, 3, 2, 5
    ex = make_experts("int8", E, S, H, F, 81)
    st, _ = make_router(E, H, k, torch.bfloat16, 82)
    need = yvf.few_workspace_bytes(N, _lib.ACT_BF16, k, ex)
    ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    x, mix = randn(83, N, H), torch.full((S,), 0.5, device="cuda")
    out = torch.full((N + 3, H), 7.0, dtype=torch.bfloat16, device="cuda")
    sh = out.clone()
    rt = yvf.Routing.empty(N, E, k, cuda)
    r, e, o = st.struct(), ex.struct(), rt.struct()
    _lib.check(_lib.lib().yvmoe_forward_few(
        x.data_ptr(), _lib.ACT_BF16, N, ctypes.byref(r), ctypes.byref(e), mix.data_ptr(), None, out.data_ptr(),
        sh.data_ptr(), ctypes.byref(o), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream), "few")
    assert bool((ws[need:] == 0xA5).all())
    assert bool((out[N:] == 7.0).all()) and bool((sh[N:] == 7.0).all())
    want = yvf.moe_forward_few(x, st, ex, mix, None)
    assert torch.equal(out[:N], want[0]) and torch.equal(sh[:N], want[1])


@pytest.mark.parametrize("fmt", ["int8", "int4"])
def test_graphs_on_one_workspace(cuda, fmt):
    """Two captured layers that share a workspace, replayed in turn with eager work between."""
    H, E, F, k, S, N = 1024, 16, 256, 4, 1, 6
    ex = make_experts(fmt, E, S, H, F, 91)
    st, _ = make_router(E, H, k, torch.bfloat16, 92)
    mix, skip = torch.ones(1, device="cuda"), randn(93, N, H)
    ws = torch.empty(yvf.few_workspace_bytes(N, _lib.ACT_BF16, k, ex), dtype=torch.uint8, device="cuda")
    xs = [randn(94, N, H), randn(95, N, H)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        yvf.moe_forward_few(xs[0], st, ex, mix, skip, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(yvf.moe_forward_few(x, st, ex, mix, skip, workspace=ws))
        graphs.append(g)
    for rep in range(4):
        for i, g in enumerate(graphs):
            xs[i].copy_(randn(100 + 2 * rep + i, N, H))
            g.replay()
            got = [t.clone() for t in (outs[i][0], outs[i][1], outs[i][2].indices, outs[i][2].weights)]
            want = yvf.moe_forward_few(xs[i], st, ex, mix, skip)
            for a, b in zip(got, (want[0], want[1], want[2].indices, want[2].weights)):
                assert torch.equal(a, b), (rep, i)


def test_calls_side_by_side(cuda):
    """Layers on several streams at once, a workspace each: the results of calls one by one."""
    H, E, F, k, S = 2048, 32, 1024, 4, 1
    ex = make_experts("int8", E, S, H, F, 101)
    st, _ = make_router(E, H, k, torch.bfloat16, 102)
    mix = torch.ones(1, device="cuda")
    xs = [randn(110 + i, 1 + 3 * i, H) for i in range(5)]
    want = [yvf.moe_forward_few(x, st, ex, mix, None)[0] for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for rep in range(3):
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(yvf.moe_forward_few(x, st, ex, mix, None)[0])
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % len(xs)]), i


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N,H,F", [(2, 512, 256), (5, 1024, 640), (16, 256, 896)])
def test_bits_do_not_go_by_the_others_choices(cuda, fmt, N, H, F):
    """A token's outputs are the same bits whatever experts the other tokens go to."""
    E, k, S = 24, 4, 1
    dt = torch.float32 if fmt == "f32" else torch.bfloat16
    ex = make_experts(fmt, E, S, H, F, 71)
    mix, x = torch.ones(1, device="cuda"), randn(72, N, H, dtype=dt)
    g = torch.Generator(device="cuda").manual_seed(73)
    w = torch.rand(N, k, device="cuda", generator=g)
    first = None
    for trial in range(4):
        idx = torch.stack([torch.randperm(E, device="cuda", generator=g)[:k] for _ in range(N)])
        if trial == 1:
            idx[:] = idx[0]  # all the same experts
        if trial == 2:
            idx[1:] = -1     # none
        idx[0] = torch.tensor([3, 7, 11, 23], device="cuda")
        out, shared, _ = yvf.experts_few(x, w, idx, ex, mix)
        if first is None:
            first = out[0].clone(), shared[0].clone()
        assert torch.equal(out[0], first[0]) and torch.equal(shared[0], first[1]), trial


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("N,E,k,S,H,F", [(16, 20, 16, 8, 128, 128), (16, 256, 16, 8, 256, 384), (9, 3, 3, 8, 640, 128)])
def test_the_most_slots(cuda, fmt, N, E, k, S, H, F):
    """As many slots, shared experts and rows of one expert as there can be."""
    print(f"most slots {fmt} {N} {E} {k} {S} {H} {F}", flush=True)
    dt = torch.float32 if fmt == "f32" else torch.bfloat16
    ex = make_experts(fmt, E, S, H, F, 81)
    g = torch.Generator(device="cuda").manual_seed(82)
    mix, x, skip = torch.rand(S, device="cuda", generator=g), randn(83, N, H, dtype=dt), randn(84, N, H, dtype=dt)
    w = torch.rand(N, k, device="cuda", generator=g)
    idx = torch.stack([torch.randperm(E, device="cuda", generator=g)[:k] for _ in range(N)])
    out, shared, invalid = yvf.experts_few(x, w, idx, ex, mix, skip)
    ref, sref, tol, stol = reference(x, w.double(), idx, ex, mix.double(), skip)
    check(out, ref, tol, "out")
    check(shared, sref, stol, "shared")
    assert int(invalid) == 0
