"""The gated feed-forward block with gradients on the host: refusals and workspace sizes."""
import ctypes
import weakref

import pytest
import torch

from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf

X, DY, WG, WU, WD, SAVED, OUT, WS, DX, DG, DU, DD = (0x10000000 * i for i in range(1, 13))
N, H, F = 100, 40, 72
ROW, MAT, KEPT = N * H * 2, H * F * 2, 2 * N * F * 4


def forward(n=N, act=_lib.ACT_BF16, h=H, f=F, x=X, wg=WG, wu=WU, wd=WD, saved=SAVED, out=OUT, ws=WS, size=None,
            weights=True):
    l = _lib.lib()
    w = _lib.SwiGLUWeights(h, f, wg, wu, wd)
    size = l.yvmoe_swiglu_workspace_bytes(n, act, h, f, 0) if size is None else size
    return l.yvmoe_swiglu_forward(x, act, n, ctypes.byref(w) if weights else None, saved, out, ws, size, None)


def backward(n=N, act=_lib.ACT_BF16, h=H, f=F, dy=DY, x=X, wg=WG, wu=WU, wd=WD, saved=SAVED, dx=DX, dg=DG, du=DU, dd=DD,
             ws=WS, size=None, weights=True):
    l = _lib.lib()
    w = _lib.SwiGLUWeights(h, f, wg, wu, wd)
    size = l.yvmoe_swiglu_workspace_bytes(n, act, h, f, 1) if size is None else size
    return l.yvmoe_swiglu_backward(dy, x, saved, act, n, ctypes.byref(w) if weights else None, dx, dg, du, dd, ws, size,
                                   None)


SIZES = [
    (dict(weights=False), _lib.YVMOE_ERR_ARG), (dict(act=9), _lib.YVMOE_ERR_DTYPE), (dict(n=-1), _lib.YVMOE_ERR_ARG),
    (dict(n=(1 << 24) + 1), _lib.YVMOE_ERR_ARG), (dict(h=0), _lib.YVMOE_ERR_SHAPE), (dict(f=0), _lib.YVMOE_ERR_SHAPE),
    (dict(h=(1 << 20) + 1), _lib.YVMOE_ERR_SHAPE), (dict(f=(1 << 20) + 1), _lib.YVMOE_ERR_SHAPE),
    (dict(n=1 << 24, h=1 << 16), _lib.YVMOE_ERR_SHAPE), (dict(n=1 << 24, f=1 << 15), _lib.YVMOE_ERR_SHAPE),
    (dict(h=1 << 20, f=1 << 19), _lib.YVMOE_ERR_SHAPE),
    (dict(wg=None), _lib.YVMOE_ERR_ARG), (dict(wu=None), _lib.YVMOE_ERR_ARG), (dict(wd=None), _lib.YVMOE_ERR_ARG),
    (dict(x=None), _lib.YVMOE_ERR_ARG), (dict(x=X + 2), _lib.YVMOE_ERR_ARG), (dict(wd=WD + 8), _lib.YVMOE_ERR_ARG),
    (dict(saved=SAVED + 4), _lib.YVMOE_ERR_ARG), (dict(ws=WS + 8), _lib.YVMOE_ERR_ARG), (dict(size=16), _lib.YVMOE_ERR_WORKSPACE),
    (dict(ws=X), _lib.YVMOE_ERR_ARG), (dict(ws=WU + MAT - 16), _lib.YVMOE_ERR_ARG), (dict(ws=SAVED), _lib.YVMOE_ERR_ARG),
]


@pytest.mark.parametrize("over,rc", SIZES + [
    (dict(out=None), _lib.YVMOE_ERR_ARG), (dict(out=OUT + 4), _lib.YVMOE_ERR_ARG), (dict(ws=None), _lib.YVMOE_ERR_ARG),
    (dict(out=X), _lib.YVMOE_ERR_ARG), (dict(out=X + ROW - 16), _lib.YVMOE_ERR_ARG), (dict(out=WG), _lib.YVMOE_ERR_ARG),
    (dict(out=SAVED + KEPT - 16), _lib.YVMOE_ERR_ARG), (dict(ws=OUT), _lib.YVMOE_ERR_ARG), (dict(saved=WD), _lib.YVMOE_ERR_ARG),
    (dict(n=0, x=None, out=None, saved=None, ws=None), _lib.YVMOE_OK),
])
def test_refused_forward(over, rc):
    assert forward(**over) == rc, _lib.lib().yvmoe_last_error()


@pytest.mark.parametrize("over,rc", SIZES + [
    (dict(dy=None), _lib.YVMOE_ERR_ARG), (dict(saved=None), _lib.YVMOE_ERR_ARG), (dict(ws=None), _lib.YVMOE_ERR_WORKSPACE),
    (dict(dx=DX + 8), _lib.YVMOE_ERR_ARG), (dict(dg=DG + 2), _lib.YVMOE_ERR_ARG), (dict(dx=X), _lib.YVMOE_ERR_ARG),
    (dict(dx=DY), _lib.YVMOE_ERR_ARG), (dict(dg=WG), _lib.YVMOE_ERR_ARG), (dict(dd=WD + MAT - 16), _lib.YVMOE_ERR_ARG),
    (dict(du=SAVED), _lib.YVMOE_ERR_ARG), (dict(dg=DU), _lib.YVMOE_ERR_ARG), (dict(dd=DX + ROW - 16), _lib.YVMOE_ERR_ARG),
    (dict(ws=DG), _lib.YVMOE_ERR_ARG),
])
def test_refused_backward(over, rc):
    assert backward(**over) == rc, _lib.lib().yvmoe_last_error()


@pytest.mark.parametrize("act", [_lib.ACT_BF16, _lib.ACT_F32])
def test_workspace_sizes(act):
    """Sizes that are refused ask for nothing; more rows never need less, over the forms' lines."""
    l = _lib.lib()
    assert l.yvmoe_swiglu_workspace_bytes(5, 9, 8, 8, 0) == 0 and l.yvmoe_swiglu_workspace_bytes(-1, act, 8, 8, 1) == 0
    assert l.yvmoe_swiglu_saved_bytes(3, 9) == 2 * 3 * 16 * 4 and l.yvmoe_swiglu_saved_bytes(0, 9) == 0
    for h, f in ((40, 72), (1000, 2731), (4096, 1408)):
        for n in (1, 32, 33, 64, 65, 1024, 1025, 5000):
            b = 4 if act == _lib.ACT_F32 else 2
            # at least h in the forward pass, h and dg, du in the backward
            assert l.yvmoe_swiglu_workspace_bytes(n, act, h, f, 0) >= n * f * b
            assert l.yvmoe_swiglu_workspace_bytes(n, act, h, f, 1) >= 3 * n * f * b


def test_refused_in_python():
    w, d = torch.zeros(8, 4), torch.zeros(4, 8)
    x = torch.zeros(3, 4)
    for call in (lambda: yvf.swiglu(x, w, w, d), lambda: yvf.swiglu(x, w, w, w), lambda: yvf.swiglu(x, w, torch.zeros(7, 4), d),
                 lambda: yvf.swiglu(torch.zeros(3, 5), w, w, d), lambda: yvf.swiglu(torch.zeros(()), w, w, d),
                 lambda: yvf.swiglu(x, w.bfloat16(), w, d), lambda: yvf.swiglu(x.half(), w.half(), w.half(), d.half()),
                 lambda: yvf.swiglu(torch.zeros(3, 0), torch.zeros(8, 0), torch.zeros(8, 0), torch.zeros(0, 8))):
        with pytest.raises(ValueError):
            call()


class _Recorded:
    """What a training call's context holds."""

    def __init__(self, stream, *leaves):
        self.stream, self.leaves = stream, {id(t) for t in leaves}


def test_captured_backward_beside_a_living_graph(monkeypatch):
    """A backward pass is not captured while a graph of the same leaves on another stream lives."""
    w, other = torch.zeros(1), torch.zeros(1)
    monkeypatch.setattr(yvf, "_training", weakref.WeakSet())
    mine, eager, same, apart = _Recorded(7, w), _Recorded(3, w, other), _Recorded(7, w), _Recorded(3, other)
    for c in (mine, same, apart):
        yvf._training.add(c)
    yvf._refuse_other_streams(mine)
    yvf._training.add(eager)
    with pytest.raises(RuntimeError, match="another stream lives"):
        yvf._refuse_other_streams(mine)
    del eager
    yvf._refuse_other_streams(mine)


def test_a_training_call_is_known_while_its_graph_lives(monkeypatch):
    """The context keeps the leaves, x's behind a view too, and is forgotten with the call's outputs."""
    monkeypatch.setattr(yvf, "_swiglu_forward", lambda x, *w: (x * 1, None))
    monkeypatch.setattr(yvf, "_stream", lambda device: 5)
    monkeypatch.setattr(yvf, "_training", weakref.WeakSet())
    x, w = torch.zeros(2, 3, 4, requires_grad=True), torch.zeros(4, 4, requires_grad=True)
    derived = w * 1
    y = yvf._SwiGLU.apply(x.view(-1, 4), w, derived, w)
    (ctx,) = yvf._training
    assert ctx.stream == 5 and ctx.leaves == {id(x), id(w)}
    del ctx, y
    assert not yvf._training


def test_what_needs_no_gradient_is_no_leaf(monkeypatch):
    """Two calls that share only an input without gradients share no leaves."""
    monkeypatch.setattr(yvf, "_swiglu_forward", lambda x, *w: (x * 1, None))
    monkeypatch.setattr(yvf, "_stream", lambda device: 5)
    monkeypatch.setattr(yvf, "_training", weakref.WeakSet())
    x, w = torch.zeros(2, 4), [torch.zeros(4, 4, requires_grad=True) for _ in range(2)]
    ys = [yvf._SwiGLU.apply(x, v, v, v) for v in w]
    assert sorted(map(sorted, (c.leaves for c in yvf._training))) == sorted([id(v)] for v in w)
    del ys
