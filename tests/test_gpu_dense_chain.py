"""The dense layers together, as a model uses them: trained, packed, served; eager, captured, on two streams."""
import pytest
import torch
import torch.nn as nn

import fp8_reference as ref
from pisceslx_amd import (YvFp8Linear, YvFp8SwiGLU, YvHybridBlockMLP, YvInt4Linear, YvRMSNorm, YvSwiGLU, pack_experts)
from pisceslx_amd import functional as yvf
from pisceslx_amd.quant import FORMAT_BY_NAME

pytestmark = pytest.mark.gpu


class Config:
    hidden_size, n_layer = 256, 4


def block(cuda, H=256, F=384, seed=0, dtype=torch.bfloat16):
    torch.manual_seed(seed)
    return YvSwiGLU(H, F, dtype=dtype).to(cuda)


def rows(cuda, n, H=256, seed=1):
    return torch.randn(n, H, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(cuda)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_training_of_the_module(cuda, dtype):
    """Gradients of a module inside torch layers, over two calls, against the same layers in 64 bits. Each gradient
    passes through at most six roundings to bf16 of independent sign (block's operands and outputs, the layer before
    and after it): 2.26e-3 sqrt(6) = 5.6e-3 in 2-norm; fp32: 1e-5 is 170 half steps."""
    m = block(cuda, dtype=dtype)
    pre, post = (nn.Linear(256, 256, bias=False, device=cuda, dtype=dtype) for _ in range(2))
    x = rows(cuda, 200).to(dtype)
    layers = [pre, m, post]
    copies = [nn.Linear(256, 256, bias=False), nn.Module(), nn.Linear(256, 256, bias=False)]
    for c, l in zip(copies, layers):
        for n, p in l.named_parameters():
            if isinstance(c, nn.Linear):
                c.weight = nn.Parameter(p.detach().cpu().double())
            else:
                setattr(c, n.replace(".", "_"), nn.Parameter(p.detach().cpu().double()))

    def exact(v):
        v = copies[0](v)
        v = nn.functional.silu(v @ copies[1].gate_proj_weight.t()) * (v @ copies[1].up_proj_weight.t())
        return copies[2](v @ copies[1].down_proj_weight.t())
    weight = rows(cuda, 200, seed=5).to(dtype)
    for part in (slice(0, 120), slice(120, 200)):  # gradients add up over two calls
        (post(m(pre(x[part]))) * weight[part]).sum().backward()
        (exact(x[part].cpu().double()) * weight[part].cpu().double()).sum().backward()
    for c, l in zip(copies, layers):
        for a, (n, b) in zip(c.parameters(), l.named_parameters()):
            rel = float((b.grad.cpu().double() - a.grad).norm() / a.grad.norm())
            print(f"{n}: {rel:.2e}", flush=True)
            assert rel <= (5.6e-3 if dtype == torch.bfloat16 else 1e-5), n


def test_no_second_derivative(cuda):
    m = block(cuda)
    x = rows(cuda, 4).requires_grad_(True)
    g, = torch.autograd.grad(m(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("n", [1, 40, 300])
def test_trained_packed_served(cuda, n):
    """A block's weights packed in 8 bits, in its own module, as an expert of a stack and from a state dict: the same
    bits, and near the block's own result: a number of four significant bits is off by 2^-4 at most, 2^-4 / sqrt(3)
    times 0.72 (the mean of 1 / mantissa) = 0.026 rms; g and u have two such roundings, 0.037, h both of theirs, g's
    times up to 1.3 by the activation's slope, 0.060, and y those of h and w_down besides: 0.071 in 2-norm, and at
    one row, 256 outputs, a quarter more."""
    m = block(cuda)
    x = rows(cuda, n)
    fp8 = YvFp8SwiGLU.from_block(m)
    out = fp8(x)
    w = (m.gate_proj.weight.detach(), m.up_proj.weight.detach(), m.down_proj.weight.detach())
    stack = pack_experts([w], 1, FORMAT_BY_NAME["fp8"], device=cuda)
    assert torch.equal(YvFp8SwiGLU.from_packed_expert(stack, 0)(x), out)
    other = YvFp8SwiGLU(256, 384, device=cuda).eval()
    other.load_reference_state_dict(m.state_dict(), "")
    assert torch.equal(other(x), out)
    with torch.no_grad():
        rel = float((out.double() - m(x).double()).norm() / m(x).double().norm())
    print(f"8 bits against bf16, {n} rows: {rel:.3f}", flush=True)
    assert rel <= 0.09


def serving(cuda):
    torch.manual_seed(3)
    qkv = YvFp8Linear.from_linear(nn.Linear(256, 256).to(cuda))
    mlp = YvFp8SwiGLU.from_block(block(cuda))
    half = YvHybridBlockMLP(Config, device=cuda, dtype=torch.bfloat16, mlp=mlp).eval()
    head = YvInt4Linear.from_linear(nn.Linear(256, 500).to(cuda), dtype=torch.bfloat16)
    norm = YvRMSNorm(256, device=cuda, dtype=torch.bfloat16)
    with torch.no_grad():
        for p in (half.norm_fusion.weight, half.norm_mlp.weight, norm.weight):
            p.uniform_(0.5, 1.5)

    def run(x):
        with torch.no_grad():
            y, loss = half(qkv(x))
            return head(norm(y)), y, loss
    return run, half, qkv


@pytest.mark.parametrize("n", [1, 7, 33, 70, 300])
def test_serving(cuda, n):
    """A projection, a block's MLP half with a dense mlp, a norm and a 4-bit head in a row; the half against its
    parts."""
    run, half, qkv = serving(cuda)
    x = rows(cuda, n)
    logits, y, loss = run(x)
    assert logits.shape == (n, 500) and float(loss) == 0 and torch.isfinite(logits).all()
    with torch.no_grad():
        h = qkv(x)
        parts = h + half.residual_scale_mlp * half.mlp(half.norm_mlp(half.norm_fusion(h)))
    assert torch.equal(parts, y)
    again = run(x)
    assert torch.equal(again[0], logits)


@pytest.mark.parametrize("n", [1, 70])
def test_serving_captured(cuda, n):
    run, _, _ = serving(cuda)
    x = rows(cuda, n)
    run(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(x)[0]
    for k in range(4):
        new = rows(cuda, n, seed=10 + k)
        x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, run(new)[0])


def test_two_streams(cuda):
    """Calls on two streams at once, each with its own workspace: the results of calls one after the other."""
    m = block(cuda, F=2000)
    fp8 = YvFp8SwiGLU.from_block(m)
    xs = [rows(cuda, 500, seed=20 + k) for k in range(2)]

    def both(x):
        with torch.no_grad():
            return m(x), fp8(x), yvf.quantize_fp8_rows(x).codes.view(torch.uint8)
    want = [both(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for s, x in zip(streams, xs):
        with torch.cuda.stream(s):
            got.append([both(x) for _ in range(4)])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for r in a:
            for u, v in zip(r, b):
                assert torch.equal(u, v)


def test_rows_once_for_several_products(cuda):
    """Rows rounded to 8 bits once and used by three projections."""
    torch.manual_seed(6)
    ps = [YvFp8Linear.from_linear(nn.Linear(256, o).to(cuda)) for o in (256, 64, 300)]
    x = rows(cuda, 90)
    q = yvf.quantize_fp8_rows(x)
    # a code times a scale takes 28 bits, so the 64-bit product is exact and fp32 rounds it once
    assert torch.equal(q.dequantize().cpu(), ref.values(*ref.rows(x.cpu()), 256).float())
    for p in ps:
        assert torch.equal(p(q), p(x))
