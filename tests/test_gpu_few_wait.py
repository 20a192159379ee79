"""The few-token kernels' wait for each other: work-groups that help, and a wait that is given up."""
import pytest
import torch

from pisceslx_amd import _lib
from pisceslx_amd import functional as yvf
from test_gpu_few import make_experts, randn

pytestmark = pytest.mark.gpu
DEFAULT, HELP, GIVE_UP = 0, 1, 2


@pytest.fixture
def set_wait(cuda):
    """How work-groups wait: HELP, GIVE_UP or DEFAULT, which it is again afterwards."""
    f = _lib.lib().yvmoe_few_set_wait
    yield f
    torch.cuda.synchronize()
    f(DEFAULT)


def problem(fmt, N, E, k, S, H, F, seed):
    dt = torch.float32 if fmt == "f32" else torch.bfloat16
    ex = make_experts(fmt, E, S, H, F, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    x, skip = randn(seed + 2, N, H, dtype=dt), randn(seed + 3, N, H, dtype=dt)
    idx = torch.stack([torch.randperm(E, device="cuda", generator=g)[:k] for _ in range(N)])
    w = torch.rand(N, k, device="cuda", generator=g)
    mix = torch.rand(S, device="cuda", generator=g) if S else None
    return lambda: yvf.experts_few(x, w, idx, ex, mix, skip)


CASES = [  # N, E, k, S, H, F
    (1, 8, 2, 1, 1024, 2816),    # two rounds of items
    (2, 6, 2, 0, 4096, 128),     # fewer items than work-groups, more columns of H
    (3, 16, 4, 2, 256, 1280),    # more items than columns of H
    (13, 40, 5, 1, 1152, 896),   # items handed out
    (16, 48, 6, 2, 2048, 1408),  # many of them, in another form of activations and h
]


@pytest.mark.parametrize("fmt", ["f32", "bf16", "int8", "int4", "fp8"])
@pytest.mark.parametrize("N,E,k,S,H,F", CASES)
def test_help(set_wait, fmt, N, E, k, S, H, F):
    """Work-groups that look once and then compute the shares that others have not marked yet: the same bits,
    though the shares' owners write them again while h is read."""
    print(f"help {fmt} {N} {E} {k} {S} {H} {F}", flush=True)
    call = problem(fmt, N, E, k, S, H, F, 1)
    want = call()
    set_wait(HELP)
    for rep in range(5):
        got = call()
        assert torch.equal(got[0], want[0]), rep
        assert S == 0 or torch.equal(got[1], want[1]), rep


@pytest.mark.parametrize("fmt", ["f32", "bf16", "int8", "int4", "fp8"])
@pytest.mark.parametrize("N,E,k,S,H,F", CASES)
def test_a_wait_given_up_shows(set_wait, fmt, N, E, k, S, H, F):
    """A work-group that gives up leaves no numbers in its columns; the last ones to end may find all of h there
    and have the right ones. The next call is as ever."""
    print(f"given up {fmt} {N} {E} {k} {S} {H} {F}", flush=True)
    call = problem(fmt, N, E, k, S, H, F, 11)
    want = call()
    set_wait(GIVE_UP)
    out, shared, _ = call()
    gone = torch.isnan(out)
    assert bool(gone.any()) and torch.equal(out[~gone], want[0][~gone])
    assert torch.equal(gone, gone[:1].expand_as(gone))  # whole columns
    if S:
        assert torch.equal(torch.isnan(shared), gone) and torch.equal(shared[~gone], want[1][~gone])
    set_wait(DEFAULT)
    got = call()
    assert torch.equal(got[0], want[0]) and (S == 0 or torch.equal(got[1], want[1]))


def test_help_in_a_graph(set_wait):
    """A captured call keeps the way of waiting it was captured with."""
    call = problem("int8", 4, 16, 4, 1, 1024, 640, 21)
    want = call()
    set_wait(HELP)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    set_wait(DEFAULT)
    for rep in range(4):
        g.replay()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), rep
        assert torch.equal(call()[0], want[0])
        torch.cuda.synchronize()
