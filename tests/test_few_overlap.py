"""The few-token entry points refuse outputs over inputs, on the host, before any GPU work: a work-group that
starts late reads x after others have written out."""
import ctypes

import pytest
import torch

from pisceslx_amd import _lib

N, E, S, H, F, K = 3, 8, 1, 128, 128, 2
X, OUT, SHARED, SKIP, MIX, WEIGHTS, INDICES, WS = (0x100000 * i for i in range(1, 9))
ROWS = N * H * 2


def call(entry, n=N, x=X, out=OUT, shared=SHARED, skip=SKIP, mix=MIX, weights=WEIGHTS, indices=INDICES, ws=WS):
    e = _lib.ExpertWeights(_lib.W_INT8, E, S, H, F, *[0x1000] * 6)
    l = _lib.lib()
    if entry == "experts":
        return l.yvmoe_experts_few(x, _lib.ACT_BF16, n, weights, _lib.ACT_F32, indices, K, ctypes.byref(e), mix, skip,
                                   out, shared, None, ws, 1 << 20, None)
    r = _lib.Router(E, H, K, 0, 1, 4, 1.0, 0x1000, 0x1000, 0x1000, 0x1000, None)
    o = _lib.Routing(*[0x1000] * 7)
    return l.yvmoe_forward_few(x, _lib.ACT_BF16, n, ctypes.byref(r), ctypes.byref(e), mix, skip, out, shared,
                               ctypes.byref(o), ws, 1 << 20, None)


def workspace_bytes():
    e = _lib.ExpertWeights(_lib.W_INT8, E, S, H, F, *[0x1000] * 6)
    return _lib.lib().yvmoe_few_workspace_bytes(N, _lib.ACT_BF16, K, ctypes.byref(e))


OVERLAPS = [
    dict(out=X), dict(out=X + ROWS - 16), dict(out=X - ROWS + 16), dict(shared=X), dict(shared=X + ROWS - 2),
    dict(ws=X), dict(ws=X + ROWS - 16), dict(x=WS + 256), dict(out=SHARED), dict(shared=OUT + 2), dict(out=WS),
    dict(shared=WS + 2), dict(mix=OUT + ROWS - 4), dict(mix=SHARED), dict(mix=WS), dict(skip=OUT + 2),
    dict(skip=SHARED - ROWS + 2), dict(skip=WS), dict(out=SKIP + 16), dict(shared=SKIP + 4),
]


@pytest.mark.parametrize("entry", ["layer", "experts"])
@pytest.mark.parametrize("over", OVERLAPS)
def test_outputs_over_inputs(entry, over):
    assert call(entry, **over) == _lib.YVMOE_ERR_ARG, over
    assert b"overlap" in _lib.lib().yvmoe_last_error()


@pytest.mark.parametrize("over", [dict(out=WEIGHTS + 16), dict(weights=SHARED), dict(indices=OUT + ROWS - 8),
                                  dict(indices=WS), dict(weights=WS + 4)])
def test_a_given_routing(over):
    assert call("experts", **over) == _lib.YVMOE_ERR_ARG, over
    assert b"overlap" in _lib.lib().yvmoe_last_error()


@pytest.mark.parametrize("entry", ["layer", "experts"])
def test_the_workspaces_last_byte(entry):
    assert call(entry, out=(WS + workspace_bytes() - 1) // 16 * 16) == _lib.YVMOE_ERR_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="the call would run on these addresses")
@pytest.mark.parametrize("entry", ["layer", "experts"])
@pytest.mark.parametrize("beside", [dict(), dict(skip=OUT), dict(skip=SHARED), dict(out=X + ROWS), dict(out=X - ROWS),
                                    dict(shared=OUT + ROWS), dict(skip=X), dict(shared=None), dict(skip=None)])
def test_neighbours_are_not_refused(entry, beside):
    """Without a GPU the launch is what fails."""
    assert call(entry, **beside) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["out", "shared"])
def test_skip_in_place(cuda, where):
    """skip as out or shared_out itself: the results of buffers apart."""
    from pisceslx_amd import functional as yvf
    from test_gpu_few import make_experts, make_router, randn
    n, e, s, h, f, k = 5, 12, 2, 640, 256, 3
    ex = make_experts("int8", e, s, h, f, 1)
    st, _ = make_router(e, h, k, torch.bfloat16, 2)
    mix, x, skip = torch.full((s,), 0.5, device="cuda"), randn(3, n, h), randn(4, n, h)
    want = yvf.moe_forward_few(x, st, ex, mix, skip)
    out, shared = torch.empty_like(x), torch.empty_like(x)
    if where == "out":
        out.copy_(skip)
        skip = out
    else:
        shared.copy_(skip)
        skip = shared
    ws = torch.empty(yvf.few_workspace_bytes(n, _lib.ACT_BF16, k, ex), dtype=torch.uint8, device="cuda")
    rt = yvf.Routing.empty(n, e, k, cuda)
    r, p, o = st.struct(), ex.struct(), rt.struct()
    _lib.check(_lib.lib().yvmoe_forward_few(
        x.data_ptr(), _lib.ACT_BF16, n, ctypes.byref(r), ctypes.byref(p), mix.data_ptr(), skip.data_ptr(), out.data_ptr(),
        shared.data_ptr(), ctypes.byref(o), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream), "few")
    assert torch.equal(out, want[0]) and torch.equal(shared, want[1])
