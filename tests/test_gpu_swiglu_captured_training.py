"""A whole training step of the block captured, its weights cast from fp32 parameters, beside a living graph of other leaves
that was recorded on another stream."""
import pytest
import torch

from pisceslx_amd import functional as yvf
from test_gpu_swiglu import make, step

pytestmark = pytest.mark.gpu


def test_step_on_cast_parameters(cuda):
    x, wg, wu, wd, dy = (t.to(cuda) for t in make(150, 136, 264, torch.bfloat16, seed=8))
    params = [torch.nn.Parameter(t.float()) for t in (wg, wu, wd)]
    other = yvf.swiglu(x, *(t.clone().requires_grad_(True) for t in (wg, wu, wd)))  # lives on the current stream

    def train():
        y = yvf.swiglu(x, *(p.to(torch.bfloat16) for p in params))
        y.backward(dy)
        return y.detach()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            train()
    torch.cuda.current_stream().wait_stream(s)
    for p in params:
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = train()
    for k in range(4):
        new = make(150, 136, 264, torch.bfloat16, seed=30 + k)
        with torch.no_grad():
            x.copy_(new[0])
            dy.copy_(new[4])
            for p, w in zip(params, new[1:4]):
                p.copy_(w.float())
        graph.replay()
        torch.cuda.synchronize()
        want = step(*new, cuda)
        assert torch.equal(y, want[0])
        for p, w in zip(params, want[2:]):
            assert torch.equal(p.grad, w.float())
    assert other.grad_fn is not None
