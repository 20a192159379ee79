"""The 4-bit linear layer on the host: storage order, quantization, refusals."""
import ctypes

import pytest
import torch

from pisceslx_amd import YvInt4Linear
from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import dequantize_int4, pack_linear, pack_linear_codes, quantize_int4, unpack_int4

P = 0x1000


@pytest.mark.parametrize("K", [1, 64, 127, 128, 200, 640])
@pytest.mark.parametrize("O", [1, 16, 37])
def test_order_of_codes(K, O):
    """Every code and scale stands where the header says."""
    groups = -(-K // 128)
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (O, groups * 64), generator=g, dtype=torch.uint8)
    scales = torch.rand(O, groups, generator=g).to(torch.bfloat16)
    pk = pack_linear_codes(codes, scales, K)
    q = unpack_int4(codes)
    for o in range(O):
        for i in range(groups * 128):
            r, c = o % 16, i % 128
            byte = 16 * (16 * (c // 32) + r) + c % 32 // 8 * 4 + c % 4
            b = int(pk.codes[o // 16, i // 128, byte])
            got = b >> 4 if c % 8 >= 4 else b & 15
            assert got == (int(q[o, i]) if i < K else 8), (o, i)
        for j in range(groups):
            assert pk.scales[o // 16, j, o % 16] == scales[o, j]
    dense = dequantize_int4(codes, scales)[:, :K]
    assert torch.equal(pk.dequantize(), dense)


def test_quantization_is_the_experts():
    w = torch.randn(48, 256, generator=torch.Generator().manual_seed(2))
    assert torch.equal(pack_linear(w).dequantize(), dequantize_int4(*quantize_int4(w)))
    odd = pack_linear(w[:, :200])
    err = (odd.dequantize() - w[:, :200]).abs()
    assert odd.dequantize().shape == (48, 200) and float(err.max()) <= float(w.abs().max()) / 7 * 0.51


@pytest.mark.parametrize("make", [
    lambda: pack_linear_codes(torch.zeros(4, 63, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.bfloat16), 128),
    lambda: pack_linear_codes(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.bfloat16), 128),
    lambda: pack_linear_codes(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.bfloat16), 128),
    lambda: pack_linear_codes(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1), 128),
    lambda: pack_linear_codes(torch.zeros(0, 64, dtype=torch.uint8), torch.zeros(0, 1, dtype=torch.bfloat16), 128),
    lambda: pack_linear(torch.zeros(8)),
])
def test_refused_weights(make):
    with pytest.raises(ValueError):
        make()


def test_refusals():
    def call(n=3, act=_lib.ACT_BF16, K=128, O=64, codes=P, scales=P, x=P, bias=P, out=P, weight=True):
        w = _lib.Int4Matrix(K, O, codes, scales)
        return _lib.lib().yvmoe_int4_linear(x, act, n, ctypes.byref(w) if weight else None, bias, out, None)

    for kw, code in [
        (dict(n=-1), _lib.YVMOE_ERR_ARG), (dict(act=5), _lib.YVMOE_ERR_DTYPE), (dict(weight=False), _lib.YVMOE_ERR_ARG),
        (dict(K=0), _lib.YVMOE_ERR_SHAPE), (dict(O=0), _lib.YVMOE_ERR_SHAPE), (dict(K=(1 << 24) + 1), _lib.YVMOE_ERR_SHAPE),
        (dict(O=(1 << 24) + 1), _lib.YVMOE_ERR_SHAPE), (dict(codes=None), _lib.YVMOE_ERR_ARG),
        (dict(scales=None), _lib.YVMOE_ERR_ARG), (dict(codes=P + 8), _lib.YVMOE_ERR_ARG),
        (dict(scales=P + 4), _lib.YVMOE_ERR_ARG), (dict(x=None), _lib.YVMOE_ERR_ARG), (dict(out=None), _lib.YVMOE_ERR_ARG),
        (dict(x=P + 1), _lib.YVMOE_ERR_ARG), (dict(out=P + 1), _lib.YVMOE_ERR_ARG), (dict(bias=P + 1), _lib.YVMOE_ERR_ARG),
        (dict(x=P + 2, act=_lib.ACT_F32), _lib.YVMOE_ERR_ARG), (dict(n=(1 << 30) + 1), _lib.YVMOE_ERR_ARG),
        (dict(n=1 << 30, O=256), _lib.YVMOE_ERR_SHAPE), (dict(n=1 << 16, O=1 << 24), _lib.YVMOE_ERR_SHAPE),
    ]:
        assert call(**kw) == code, kw
        assert _lib.lib().yvmoe_last_error()
    assert call(n=0, x=None, out=None) == _lib.YVMOE_OK
    for out in (P, P + 3 * 128 * 2 - 2, P - 3 * 64 * 2 + 2):  # over x, its last element, its first
        assert call(x=P, out=out) == _lib.YVMOE_ERR_ARG
        assert b"overlaps" in _lib.lib().yvmoe_last_error()


def test_refused_tensors():
    pk = pack_linear(torch.randn(16, 128))
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    for bad in (lambda: yvf.int4_linear(x, pk), lambda: yvf.int4_linear(x[:, :64], pk),
                lambda: yvf.int4_linear(torch.zeros((), dtype=torch.bfloat16), pk)):
        with pytest.raises(ValueError):
            bad()


def test_module():
    dense = torch.nn.Linear(200, 33)
    m = YvInt4Linear.from_linear(dense)
    pk = pack_linear(dense.weight.detach())
    assert torch.equal(m.packed.dequantize(), pk.dequantize()) and torch.equal(m.bias, dense.bias)
    other = YvInt4Linear(200, 33).to(torch.bfloat16)  # a change of dtype: the bias alone
    assert other.bias.dtype == torch.bfloat16 and other.packed.scales.dtype == torch.bfloat16
    other.load_state_dict(m.state_dict())
    assert torch.equal(other.packed.dequantize(), pk.dequantize())
    assert torch.equal(other.bias, dense.bias.detach().to(torch.bfloat16))
    with pytest.raises(NotImplementedError):
        other.train()(torch.zeros(1, 200))
    with pytest.raises(ValueError):
        m(torch.zeros(1, 200))  # no CPU form
    with pytest.raises(ValueError):
        m.set_weight(pack_linear(torch.zeros(33, 201)))
    with pytest.raises(ValueError):
        YvInt4Linear(0, 33)
    assert float(YvInt4Linear(130, 17).packed.dequantize().abs().max()) == 0


def test_module_from_a_reference_state():
    w, b = torch.randn(40, 256), torch.randn(40)
    q = (w / (w.abs().amax(dim=0, keepdim=True) / 127)).round().to(torch.int8)
    scale, zero = w.abs().amax(dim=0, keepdim=True) / 127, torch.zeros(1, 256)
    m = YvInt4Linear(256, 40)
    m.load_reference_state_dict({"a.proj.weight": w, "a.proj.bias": b}, "a.proj")
    assert torch.equal(m.packed.codes, pack_linear(w).codes) and torch.equal(m.bias.detach(), b)
    m.load_reference_state_dict({"p.q_weight": q, "p.scale": scale, "p.zero_point": zero, "p.bias": b}, "p")
    assert torch.equal(m.packed.codes, pack_linear(q.float() * scale).codes)
    with pytest.raises(KeyError):
        m.load_reference_state_dict({"p.weight": w}, "p")
