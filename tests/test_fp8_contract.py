"""8-bit rows, linear layer and gated block on the host: storage order, quantization, refusals, modules."""
import ctypes

import pytest
import torch

import fp8_reference as ref
from pisceslx_amd import YvFp8Linear, YvFp8SwiGLU, YvHybridBlockMLP, YvSwiGLU
from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf
from pisceslx_amd import quant

# addresses of tensors far from each other
X, CODES, SCALES, BIAS, OUT, WS, XS = (0x10000000 * i for i in range(1, 8))


@pytest.mark.parametrize("K", [1, 64, 127, 128, 200, 384])
@pytest.mark.parametrize("O", [1, 16, 37, 130])
def test_order_of_codes(K, O):
    """Every code and scale stands where the header says."""
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (O, K), generator=g, dtype=torch.uint8)
    scales = torch.rand(-(-O // 128), -(-K // 128), generator=g)
    pk = quant.pack_fp8_linear_codes(codes, scales, K)
    flat = pk.codes.view(-(-O // 16), -1, 1024)
    for o in range(-(-O // 16) * 16):
        for i in range(-(-K // 128) * 128):
            byte = 16 * (16 * (i % 64 // 16) + o % 16) + i % 16
            assert int(flat[o // 16, i // 64, byte]) == (int(codes[o, i]) if o < O and i < K else 0)
    assert torch.equal(pk.scales, scales)
    bytes_as_float = quant.pack_fp8_linear_codes(codes.view(torch.float8_e4m3fn), scales, K)
    assert torch.equal(bytes_as_float.codes, pk.codes)


def test_dequantized():
    q = torch.randn(70, 200, generator=torch.Generator().manual_seed(2)).mul_(100).to(torch.float8_e4m3fn)
    s = torch.rand(1, 2) + 0.5
    assert torch.equal(quant.pack_fp8_linear_codes(q, s, 200).dequantize().double(),
                       ref.weight(q.view(torch.uint8), s).float().double())


@pytest.mark.parametrize("O,K", [(128, 256), (100, 300), (1, 1)])
def test_quantization_of_weights(O, K):
    w = torch.randn(O, K, generator=torch.Generator().manual_seed(3))
    d = quant.pack_fp8_linear(w).dequantize()
    # half a step of three mantissa bits, or of the smallest exponent's
    top = float(w.abs().max())
    assert d.shape == w.shape and bool(((d - w).abs() <= w.abs() * 2.0 ** -4 + top / 448 * 2.0 ** -10).all())


@pytest.mark.parametrize("make", [
    lambda: quant.pack_fp8_linear_codes(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(1, 1), 64),
    lambda: quant.pack_fp8_linear_codes(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1, 1), 63),
    lambda: quant.pack_fp8_linear_codes(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(2, 1), 64),
    lambda: quant.pack_fp8_linear_codes(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1, 1).bfloat16(), 64),
    lambda: quant.pack_fp8_linear_codes(torch.zeros(0, 64, dtype=torch.uint8), torch.zeros(0, 1), 64),
    lambda: quant.pack_fp8_linear_codes(torch.zeros(4, 0, dtype=torch.uint8), torch.zeros(1, 0), 0),
    lambda: quant.pack_fp8_linear_codes(torch.zeros(256, dtype=torch.uint8), torch.zeros(1, 1), 64),
    lambda: quant.pack_fp8_linear(torch.zeros(8)),
    lambda: quant.Fp8Rows(200, torch.zeros(3, 200, dtype=torch.float8_e4m3fn), torch.zeros(2, 3)),
    lambda: quant.Fp8Rows(200, torch.zeros(3, 256, dtype=torch.uint8), torch.zeros(2, 3)),
    lambda: quant.Fp8Rows(200, torch.zeros(3, 256, dtype=torch.float8_e4m3fn), torch.zeros(3, 2)),
    lambda: quant.Fp8Rows(0, torch.zeros(3, 0, dtype=torch.float8_e4m3fn), torch.zeros(0, 3)),
])
def test_refused_weights_and_rows(make):
    with pytest.raises(ValueError):
        make()


def rows_call(x=X, act=_lib.ACT_BF16, n=5, k=300, codes=CODES, scales=SCALES):
    return _lib.lib().yvmoe_quantize_fp8_rows(x, act, n, k, codes, scales, None)


@pytest.mark.parametrize("over,rc", [
    (dict(act=7), _lib.YVMOE_ERR_DTYPE), (dict(n=-1), _lib.YVMOE_ERR_ARG), (dict(n=(1 << 24) + 1), _lib.YVMOE_ERR_ARG),
    (dict(k=0), _lib.YVMOE_ERR_SHAPE), (dict(k=(1 << 20) + 1), _lib.YVMOE_ERR_SHAPE), (dict(x=None), _lib.YVMOE_ERR_ARG),
    (dict(codes=None), _lib.YVMOE_ERR_ARG), (dict(scales=None), _lib.YVMOE_ERR_ARG), (dict(x=X + 1), _lib.YVMOE_ERR_ARG),
    (dict(act=_lib.ACT_F32, x=X + 2), _lib.YVMOE_ERR_ARG), (dict(codes=CODES + 8), _lib.YVMOE_ERR_ARG),
    (dict(scales=SCALES + 2), _lib.YVMOE_ERR_ARG), (dict(codes=X), _lib.YVMOE_ERR_ARG),
    (dict(scales=X + 5 * 300 * 2 - 4), _lib.YVMOE_ERR_ARG), (dict(scales=CODES + 5 * 384 - 4), _lib.YVMOE_ERR_ARG),
    (dict(n=0, x=None, codes=None, scales=None), _lib.YVMOE_OK),
])
def test_refused_rows(over, rc):
    assert rows_call(**over) == rc, _lib.lib().yvmoe_last_error()


def linear_call(n=5, K=300, O=40, codes=CODES, scales=SCALES, x=X, bias=BIAS, out=OUT, ws=WS, size=None, weight=True,
                xs=None):
    l = _lib.lib()
    w = _lib.Fp8Matrix(K, O, codes, scales)
    p = ctypes.byref(w) if weight else None
    if xs is None:
        size = l.yvmoe_fp8_linear_workspace_bytes(max(n, 1), max(K, 1), max(O, 1)) if size is None else size
        return l.yvmoe_fp8_linear(x, n, p, bias, out, ws, size, None)
    size = l.yvmoe_fp8_linear_rows_workspace_bytes(max(n, 1), max(K, 1), max(O, 1)) if size is None else size
    return l.yvmoe_fp8_linear_rows(x, xs, n, p, bias, out, ws, size, None)


LINEAR = [
    (dict(weight=False), _lib.YVMOE_ERR_ARG), (dict(n=-1), _lib.YVMOE_ERR_ARG), (dict(n=(1 << 24) + 1), _lib.YVMOE_ERR_ARG),
    (dict(K=0), _lib.YVMOE_ERR_SHAPE), (dict(O=0), _lib.YVMOE_ERR_SHAPE), (dict(K=(1 << 20) + 1), _lib.YVMOE_ERR_SHAPE),
    (dict(O=(1 << 20) + 1), _lib.YVMOE_ERR_SHAPE), (dict(n=1 << 24, O=1 << 13), _lib.YVMOE_ERR_SHAPE),
    (dict(codes=None), _lib.YVMOE_ERR_ARG), (dict(scales=None), _lib.YVMOE_ERR_ARG), (dict(x=None), _lib.YVMOE_ERR_ARG),
    (dict(out=None), _lib.YVMOE_ERR_ARG), (dict(codes=CODES + 8), _lib.YVMOE_ERR_ARG),
    (dict(scales=SCALES + 2), _lib.YVMOE_ERR_ARG), (dict(x=X + 1), _lib.YVMOE_ERR_ARG), (dict(bias=BIAS + 1), _lib.YVMOE_ERR_ARG),
    (dict(out=OUT + 2), _lib.YVMOE_ERR_ARG), (dict(out=X), _lib.YVMOE_ERR_ARG), (dict(out=BIAS), _lib.YVMOE_ERR_ARG),
    (dict(out=CODES + 3 * 3 * 2048 - 8), _lib.YVMOE_ERR_ARG), (dict(scales=OUT + 396), _lib.YVMOE_ERR_ARG),
    (dict(n=0, x=None, out=None, bias=None), _lib.YVMOE_OK),
]


@pytest.mark.parametrize("over,rc", LINEAR + [
    (dict(ws=None), _lib.YVMOE_ERR_ARG), (dict(ws=WS + 8), _lib.YVMOE_ERR_ARG), (dict(size=100), _lib.YVMOE_ERR_WORKSPACE),
    (dict(ws=X), _lib.YVMOE_ERR_ARG), (dict(ws=CODES), _lib.YVMOE_ERR_ARG), (dict(ws=OUT), _lib.YVMOE_ERR_ARG),
])
def test_refused_linear(over, rc):
    assert linear_call(**over) == rc, _lib.lib().yvmoe_last_error()


@pytest.mark.parametrize("over,rc", LINEAR + [
    (dict(xs=0), _lib.YVMOE_ERR_ARG), (dict(x=X + 8), _lib.YVMOE_ERR_ARG), (dict(xs=XS + 2), _lib.YVMOE_ERR_ARG),
    (dict(out=XS), _lib.YVMOE_ERR_ARG),
    # a contraction that is split needs a workspace
    (dict(n=70, K=8192, O=512, ws=None), _lib.YVMOE_ERR_WORKSPACE),
    (dict(n=70, K=8192, O=512, size=100), _lib.YVMOE_ERR_WORKSPACE), (dict(n=70, K=8192, O=512, ws=OUT), _lib.YVMOE_ERR_ARG),
])
def test_refused_linear_rows(over, rc):
    assert linear_call(**dict(dict(xs=XS), **over)) == rc, _lib.lib().yvmoe_last_error()


def block_call(n=5, gate=(300, 200), up=(300, 200), down=(200, 300), x=X, out=OUT, ws=WS, size=None, codes=CODES):
    l = _lib.lib()
    ms = [_lib.Fp8Matrix(i, o, codes + 0x1000000 * k, SCALES + 0x1000000 * k) for k, (i, o) in enumerate((gate, up, down))]
    size = l.yvmoe_fp8_swiglu_workspace_bytes(n, *gate) if size is None else size
    return l.yvmoe_fp8_swiglu(x, n, *map(ctypes.byref, ms), out, ws, size, None)


@pytest.mark.parametrize("over,rc", [
    (dict(n=-1), _lib.YVMOE_ERR_ARG), (dict(up=(300, 201)), _lib.YVMOE_ERR_SHAPE), (dict(up=(301, 200)), _lib.YVMOE_ERR_SHAPE),
    (dict(down=(200, 301)), _lib.YVMOE_ERR_SHAPE), (dict(down=(300, 200)), _lib.YVMOE_ERR_SHAPE), (dict(x=None), _lib.YVMOE_ERR_ARG),
    (dict(out=None), _lib.YVMOE_ERR_ARG), (dict(ws=None), _lib.YVMOE_ERR_ARG), (dict(size=64), _lib.YVMOE_ERR_WORKSPACE),
    (dict(x=X + 1), _lib.YVMOE_ERR_ARG), (dict(out=OUT + 4), _lib.YVMOE_ERR_ARG), (dict(ws=WS + 8), _lib.YVMOE_ERR_ARG),
    (dict(out=X), _lib.YVMOE_ERR_ARG), (dict(ws=X), _lib.YVMOE_ERR_ARG), (dict(ws=OUT), _lib.YVMOE_ERR_ARG),
    (dict(out=CODES + 0x2000000), _lib.YVMOE_ERR_ARG), (dict(ws=SCALES + 0x1000000), _lib.YVMOE_ERR_ARG),
    (dict(n=0, x=None, out=None, ws=None), _lib.YVMOE_OK),
])
def test_refused_block(over, rc):
    assert block_call(**over) == rc, _lib.lib().yvmoe_last_error()


def test_refused_in_python():
    w = quant.pack_fp8_linear(torch.randn(40, 72))
    bf = torch.zeros(3, 72, dtype=torch.bfloat16)
    for call in (lambda: yvf.fp8_linear(bf, w), lambda: yvf.fp8_linear(torch.zeros(3, 71, dtype=torch.bfloat16), w),
                 lambda: yvf.fp8_linear(torch.zeros(3, 72), w), lambda: yvf.fp8_linear(torch.zeros((), dtype=torch.bfloat16), w),
                 lambda: yvf.quantize_fp8_rows(bf), lambda: yvf.quantize_fp8_rows(torch.zeros(3, 0)),
                 lambda: yvf.fp8_linear(quant.Fp8Rows(80, torch.zeros(3, 128, dtype=torch.float8_e4m3fn), torch.zeros(1, 3)), w),
                 lambda: yvf.fp8_swiglu(bf, w, w, w),
                 lambda: yvf.fp8_swiglu(torch.zeros(3, 72), w, w, quant.pack_fp8_linear(torch.randn(72, 40)))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError, match="gradient"):
        yvf.fp8_linear(bf.clone().requires_grad_(True), w)


def test_linear_module():
    g = torch.Generator().manual_seed(4)
    w, b = torch.randn(40, 200, generator=g), torch.randn(40, generator=g)
    m = YvFp8Linear(200, 40)
    before = m.codes.clone()
    with pytest.raises(KeyError):
        m.load_reference_state_dict({"p.weight": w}, "p")
    assert torch.equal(m.codes, before)
    m.load_reference_state_dict({"p.weight": w, "p.bias": b}, "p")
    assert torch.equal(m.packed.dequantize(), quant.pack_fp8_linear(w).dequantize())
    assert torch.equal(m.bias, b.to(torch.bfloat16))
    with pytest.raises(ValueError, match="p.bias"):
        YvFp8Linear(200, 40, bias=False).load_reference_state_dict({"p.weight": w, "p.bias": b}, "p")
    again = YvFp8Linear(200, 40)
    again.load_state_dict(m.state_dict())
    moved = again.to(torch.bfloat16)  # a change of dtype leaves the scales alone
    assert torch.equal(moved.packed.dequantize(), m.packed.dequantize())
    with pytest.raises(NotImplementedError):
        m.train()(torch.zeros(1, 200, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        m.set_weight(quant.pack_fp8_linear(torch.randn(40, 100)))
    with pytest.raises(ValueError):
        YvFp8Linear(200, 40, dtype=torch.float32)


def test_block_modules():
    block = YvSwiGLU(64, 96)
    assert sorted(block.state_dict()) == ["down_proj.weight", "gate_proj.weight", "up_proj.weight"]
    fp8 = YvFp8SwiGLU.from_block(block)
    other = YvFp8SwiGLU(64, 96).eval()
    other.load_reference_state_dict({"e.3." + k: v for k, v in block.state_dict().items()}, "e.3.")
    for a, b, n in zip(fp8.packed(), other.packed(), ("gate_proj", "up_proj", "down_proj")):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        assert torch.equal(a.dequantize(), quant.pack_fp8_linear(getattr(block, n).weight.detach()).dequantize())
    with pytest.raises(NotImplementedError):
        fp8.train()(torch.zeros(1, 64, dtype=torch.bfloat16))
    mats = [tuple(torch.randn(*s) for s in ((128, 256), (128, 256), (256, 128))) for _ in range(3)]
    pk = quant.pack_experts(mats, 2, _lib.W_FP8)
    e = YvFp8SwiGLU.from_packed_expert(pk, 2)
    assert e.gate_proj.codes.data_ptr() == pk.w_gate[2].data_ptr()
    for p, w in zip(e.packed(), mats[2]):
        assert torch.equal(p.dequantize(), quant.pack_fp8_linear(w).dequantize())
    for bad in (lambda: YvFp8SwiGLU.from_packed_expert(pk, 3), lambda: YvSwiGLU(0, 8),
                lambda: YvFp8SwiGLU.from_packed_expert(quant.pack_experts(mats, 2, _lib.W_BF16), 0)):
        with pytest.raises(ValueError):
            bad()

    class Cfg:
        hidden_size, n_layer = 32, 4
    with pytest.raises(ValueError, match="hidden_size"):
        YvHybridBlockMLP(Cfg, mlp=block)
