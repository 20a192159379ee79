"""The few-token form inside the layers, 4-bit linear layers, and a block of them, captured and
replayed, against plain statements in 64 bits."""
import pytest
import torch

from pisceslx_amd import YvDeepSeekMoELayer, YvHybridBlockMLP, YvInt4Linear
from pisceslx_amd.quant import pack_linear
from test_gpu_few import check, randn, reference
from test_gpu_int4_linear import check as check_linear
from test_gpu_module import Cfg, moegate_state_dict, reference_state_dict

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def make_layer(router, fmt, few_tokens, shared=2, dtype=BF16):
    cfg = Cfg()
    cfg.moe_shared_experts = shared
    layer = YvDeepSeekMoELayer(cfg, device="cuda", dtype=dtype, weight_format=fmt, router=router,
                               few_tokens=few_tokens).eval()
    sd = reference_state_dict(cfg)
    if router == "moegate":
        sd = {k: v for k, v in sd.items() if not k.startswith("router.")}
        sd.update(moegate_state_dict(cfg))
    layer.load_reference_state_dict(sd, strict=router == "moegate")
    return layer


def check_layer(layer, x, out, skip, what):
    x2d = x.reshape(-1, x.shape[-1])
    r = layer.last_routing
    mix = layer._mix()
    ref, shared, tol, stol = reference(x2d, r.weights.double(), r.indices, layer.experts_packed,
                                       None if mix is None else mix.double(),
                                       None if skip is None else skip.reshape(x2d.shape))
    check(out.reshape(x2d.shape), ref, tol, what)
    if layer.num_shared_experts:
        check(layer._skip_buffer.reshape(x2d.shape), shared, stol, what + " shared")


@pytest.mark.parametrize("fmt,dtype", [("int8", BF16), ("int4", BF16), ("bf16", BF16), ("f32", torch.float32)])
@pytest.mark.parametrize("router", ["stable", "moegate"])
@pytest.mark.parametrize("B,S", [(1, 1), (3, 2), (16, 1)])
def test_layer(cuda, router, fmt, dtype, B, S):
    print(f"few-token layer {router} {fmt} {B} x {S}", flush=True)
    layer = make_layer(router, fmt, 16, dtype=dtype)
    general = make_layer(router, fmt, 0, dtype=dtype)
    if router == "moegate":
        layer.router._path_moe_stage_size = general.router._path_moe_stage_size = 1
    skip = None
    for call in range(3):  # from the second on with the skip residual of the one before
        x = randn(30 + call, B, S, layer.hidden_size, dtype=dtype)
        out, loss = layer(x)
        check_layer(layer, x, out, skip, f"call {call}")
        _, general_loss = general(x)
        if router == "moegate":
            assert torch.equal(layer.last_routing.indices, general.last_routing.indices)
            assert torch.equal(layer.last_routing.weights, general.last_routing.weights)
        assert torch.equal(loss, general_loss) and loss.dtype == general_loss.dtype
        skip = layer._skip_buffer.clone()


def test_longer_calls_are_as_before(cuda):
    few, general = make_layer("stable", "int8", 4), make_layer("stable", "int8", 0)
    for n in (5, 3, 40):
        x = randn(n, 1, n, few.hidden_size)
        a, b = few(x)[0], general(x)[0]
        assert n <= 4 or torch.equal(a, b)
        few._skip_buffer = general._skip_buffer = None


def test_stage_cache(cuda):
    """Later calls of a stage take the first one's routing, also when the general form made it."""
    layer = make_layer("moegate", "bf16", 16, shared=0)
    assert layer.router._path_moe_stage_size == 4
    first = None
    for i in range(6):
        layer.few_tokens = 0 if i == 0 else 16
        x = randn(50 + i, 2, 4, layer.hidden_size)
        out, _ = layer(x)
        if i % 4 == 0:
            first = layer.last_routing.indices.clone()
        assert torch.equal(layer.last_routing.indices, first)
        check_layer(layer, x, out, None, f"call {i}")


def test_linear_module(cuda):
    dense = torch.nn.Linear(300, 77, device="cuda")
    m = YvInt4Linear.from_linear(dense, dtype=BF16)
    pk = pack_linear(dense.weight.detach())
    assert torch.equal(m.codes, pk.codes) and torch.equal(m.packed.scales, pk.scales)
    x = randn(60, 4, 5, 600)[..., ::2]  # not contiguous
    check_linear(x.reshape(-1, 300), pk, m.bias, m(x).reshape(-1, 77), "module")
    fp = YvInt4Linear.from_linear(dense).to("cpu").cuda()
    xf = randn(61, 4, 300, dtype=torch.float32)
    check_linear(xf, pk, fp.bias, fp(xf), "fp32")
    with pytest.raises(ValueError):
        m(xf)  # a bias of another type


@pytest.mark.parametrize("tokens", [1, 5, 16])
def test_a_block_between_linear_layers(cuda, tokens):
    """A projection, the block's MoE half in its few-token form and a projection: step by step against
    64 bits, then captured and replayed between eager calls of the same modules."""
    class BlockCfg(Cfg):
        n_layer = 4
        moe_few_tokens = 16
    cfg = BlockCfg()
    torch.manual_seed(3)
    H = cfg.hidden_size
    block = YvHybridBlockMLP(cfg, device="cuda", dtype=BF16, weight_format="int8").eval()
    assert block.mlp.few_tokens == 16
    sd = {k: v for k, v in reference_state_dict(cfg).items() if not k.startswith("router.")}
    sd.update(moegate_state_dict(cfg))
    block.mlp.load_reference_state_dict(sd, strict=True)
    block.mlp.router._path_moe_stage_size = 1
    first = YvInt4Linear.from_linear(torch.nn.Linear(520, H, device="cuda", dtype=BF16))
    last = YvInt4Linear.from_linear(torch.nn.Linear(H, 1003, bias=False, device="cuda", dtype=BF16))
    seen = {}
    block.mlp.register_forward_hook(lambda m, args, res: seen.update(x=args[0], out=res[0]))

    @torch.no_grad()
    def run(x):
        block.mlp._skip_buffer = None
        h = first(x)
        b, _ = block(h)
        return h, b, last(b)

    x = randn(70, 1, tokens, 520)
    h, b, y = run(x)
    check_linear(x[0], first.packed, first.bias, h[0], "first")
    check_layer(block.mlp, seen["x"], seen["out"], None, "block")
    check_linear(b[0], last.packed, None, y[0], "last")
    # captured on a stream of its own, with a workspace of its own
    static = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block.mlp._workspace = None
        run(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(static)[2]
    held, block.mlp._workspace = block.mlp._workspace, None  # the graph's
    for i in range(4):
        xi = randn(80 + i, 1, tokens, 520)
        want = run(xi)[2]
        static.copy_(xi)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want), i
    del held
