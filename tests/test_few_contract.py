"""Refusals of the few-token layer's entry points: checked on the host, before any GPU work."""
import ctypes

import pytest
import torch

from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import pack_experts

P = 0x1000  # an aligned address that a refused call never reads


def _experts(fmt=_lib.W_INT8, E=8, S=1, H=128, F=128, **over):
    v = dict(w_gate=P, w_up=P, w_down=P, s_gate=P, s_up=P, s_down=P)
    v.update(over)
    return _lib.ExpertWeights(fmt, E, S, H, F, *v.values())


def _router(E=8, H=128, k=2, fixed=0, dynamic=1, w=P, b1=P):
    return _lib.Router(E, H, k, fixed, dynamic, 4, 1.0, w, b1, P, P, None)


def _routing(**over):
    v = dict(weights=P, indices=P, counts=P, offsets=P, perm=P, pos=P, capacity=P)
    v.update(over)
    return _lib.Routing(*v.values())


def _forward(n=3, act=_lib.ACT_BF16, router=None, experts=None, routing=None, x=P, out=P, mix=P, ws=P, nbytes=1 << 30):
    r, e, o = router or _router(), experts or _experts(), routing or _routing()
    return _lib.lib().yvmoe_forward_few(x, act, n, ctypes.byref(r), ctypes.byref(e), mix, None, out, None,
                                        ctypes.byref(o), ws, nbytes, None)


def _given(n=3, act=_lib.ACT_BF16, k=2, wdt=_lib.ACT_F32, experts=None, w=P, idx=P, x=P, out=P, mix=P, ws=P,
           nbytes=1 << 30):
    e = experts or _experts()
    return _lib.lib().yvmoe_experts_few(x, act, n, w, wdt, idx, k, ctypes.byref(e), mix, None, out, None, None, ws,
                                        nbytes, None)


def test_sizes():
    l = _lib.lib()
    e = _experts(E=64, S=2, H=4096, F=1408)
    sizes = [l.yvmoe_few_workspace_bytes(n, _lib.ACT_BF16, 6, ctypes.byref(e)) for n in range(17)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    assert sizes[16] >= 16 * 8 * 1408 * 2
    assert l.yvmoe_few_workspace_bytes(17, _lib.ACT_BF16, 6, ctypes.byref(e)) == 0
    assert l.yvmoe_few_workspace_bytes(-1, _lib.ACT_BF16, 6, ctypes.byref(e)) == 0
    assert l.yvmoe_few_workspace_bytes(1, _lib.ACT_BF16, 17, ctypes.byref(e)) == 0
    assert l.yvmoe_few_workspace_bytes(1, _lib.ACT_F32, 6, ctypes.byref(e)) == 0  # int8 needs bf16


@pytest.mark.parametrize("call", [_forward, _given])
def test_refusals_of_both(call):
    small = _lib.lib().yvmoe_few_workspace_bytes(3, _lib.ACT_BF16, 2, ctypes.byref(_experts())) - 1
    for kw, code in [
        (dict(n=17), _lib.YVMOE_ERR_SHAPE), (dict(n=-1), _lib.YVMOE_ERR_ARG), (dict(act=7), _lib.YVMOE_ERR_DTYPE),
        (dict(act=_lib.ACT_F32), _lib.YVMOE_ERR_DTYPE), (dict(x=None), _lib.YVMOE_ERR_ARG),
        (dict(out=None), _lib.YVMOE_ERR_ARG), (dict(x=P + 2), _lib.YVMOE_ERR_ARG), (dict(out=P + 8), _lib.YVMOE_ERR_ARG),
        (dict(ws=P + 8), _lib.YVMOE_ERR_ARG), (dict(ws=None), _lib.YVMOE_ERR_WORKSPACE),
        (dict(nbytes=small), _lib.YVMOE_ERR_WORKSPACE), (dict(mix=None), _lib.YVMOE_ERR_ARG),
        (dict(experts=_experts(fmt=9)), _lib.YVMOE_ERR_DTYPE), (dict(experts=_experts(H=96)), _lib.YVMOE_ERR_SHAPE),
        (dict(experts=_experts(fmt=_lib.W_INT4, F=192)), _lib.YVMOE_ERR_SHAPE),
        (dict(experts=_experts(S=9)), _lib.YVMOE_ERR_SHAPE), (dict(experts=_experts(E=257)), _lib.YVMOE_ERR_SHAPE),
        (dict(experts=_experts(w_up=None)), _lib.YVMOE_ERR_ARG), (dict(experts=_experts(s_down=None)), _lib.YVMOE_ERR_ARG),
        (dict(experts=_experts(w_down=P + 8)), _lib.YVMOE_ERR_ARG), (dict(experts=_experts(s_up=P + 2)), _lib.YVMOE_ERR_ARG),
    ]:
        assert call(**kw) == code, kw
        assert _lib.lib().yvmoe_last_error()


def test_refusals_of_the_layer():
    for kw, code in [
        (dict(router=_router(E=9)), _lib.YVMOE_ERR_SHAPE), (dict(router=_router(H=256)), _lib.YVMOE_ERR_SHAPE),
        (dict(router=_router(k=9)), _lib.YVMOE_ERR_SHAPE), (dict(router=_router(w=None)), _lib.YVMOE_ERR_ARG),
        (dict(router=_router(w=P + 8)), _lib.YVMOE_ERR_ARG), (dict(router=_router(b1=None)), _lib.YVMOE_ERR_ARG),
        (dict(routing=_routing(perm=None)), _lib.YVMOE_ERR_ARG),
        (dict(routing=_routing(capacity=None)), _lib.YVMOE_ERR_ARG),
    ]:
        assert _forward(**kw) == code, kw


def test_refusals_of_a_given_routing():
    for kw, code in [(dict(k=0), _lib.YVMOE_ERR_SHAPE), (dict(k=17), _lib.YVMOE_ERR_SHAPE),
                     (dict(wdt=3), _lib.YVMOE_ERR_DTYPE), (dict(w=None), _lib.YVMOE_ERR_ARG),
                     (dict(idx=None), _lib.YVMOE_ERR_ARG)]:
        assert _given(**kw) == code, kw


def test_cpu_tensors_are_refused():
    ex = pack_experts([(torch.zeros(64, 64), torch.zeros(64, 64), torch.zeros(64, 64))], 1, _lib.W_BF16)
    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        yvf.experts_few(x, torch.ones(1, 1), torch.zeros(1, 1, dtype=torch.int64), ex)


def test_layer_argument():
    from pisceslx_amd import YvDeepSeekMoELayer

    class Cfg:
        hidden_size = 64
        intermediate_size = 64
        moe_num_experts = 4
        moe_top_k = 2
    assert YvDeepSeekMoELayer(Cfg(), router="stable").few_tokens == 0
    assert YvDeepSeekMoELayer(Cfg(), router="stable", few_tokens=16).few_tokens == 16
    Cfg.moe_few_tokens = 5
    assert YvDeepSeekMoELayer(Cfg(), router="stable").few_tokens == 5
    assert YvDeepSeekMoELayer(Cfg(), router="stable", few_tokens=0).few_tokens == 0
    for bad in (-1, 17):
        with pytest.raises(ValueError):
            YvDeepSeekMoELayer(Cfg(), router="stable", few_tokens=bad)


def test_lazy_routing():
    r, e = yvf.Routing.lazy(3, 100, 4, "cpu"), yvf.Routing.empty(3, 100, 4, "cpu")
    o = r.struct()
    for name in ("weights", "indices", "counts", "offsets", "perm", "pos", "capacity"):
        a, b = getattr(r, name), getattr(e, name)
        assert a.shape == b.shape and a.dtype == b.dtype and a.is_contiguous()
        assert a.data_ptr() == getattr(o, name) and getattr(r, name) is a
    assert isinstance(r, yvf.Routing)
    with pytest.raises(AttributeError):
        r.other
