"""A captured layer call and longer eager calls of the same layer: the graph keeps the memory it writes to."""
import pytest
import torch

from test_gpu_few import randn
from test_gpu_few_module import make_layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("router,few", [("stable", 16), ("moegate", 0), ("moegate", 16)])
def test_a_longer_call_after_the_capture(cuda, router, few):
    layer = make_layer(router, "int8", few, shared=0)
    if router == "moegate":
        layer.router._path_moe_stage_size = 1
    x = randn(1, 1, 1, layer.hidden_size)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x)  # leaves a workspace with the layer
    torch.cuda.current_stream().wait_stream(side)
    kept = layer._workspace
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = layer(x)
    assert layer._workspace is kept  # not the graph's
    kept = None
    layer(randn(2, 1, 16, layer.hidden_size))  # takes a larger one
    layer(randn(3, 1, 300, layer.hidden_size))
    torch.cuda.synchronize()
    # whatever the longer calls have freed
    held = [torch.full((n,), 0x5A, dtype=torch.uint8, device="cuda") for n in [1 << i for i in range(9, 23)] * 6]
    for rep in range(4):
        x.copy_(randn(10 + rep, 1, 1, layer.hidden_size))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert all(bool((t == 0x5A).all()) for t in held), rep
        assert torch.equal(got, layer(x)[0]), rep
