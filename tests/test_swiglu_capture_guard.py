"""The refusal of a captured backward pass beside a living graph of the same leaves, with torch's own graphs and the
native calls replaced: on the CPU."""
import sys
import threading
import weakref

import pytest
import torch

from pisceslx_amd import functional as yvf


@pytest.fixture
def captured(monkeypatch):
    """Calls record the stream that is set here, every backward pass counts as captured, and nothing is launched."""
    stream = [0]
    monkeypatch.setattr(yvf, "_swiglu_forward", lambda x, *w: (x * 1, torch.zeros(1)))
    monkeypatch.setattr(yvf, "_stream", lambda device: stream[0])
    monkeypatch.setattr(yvf, "_launch", lambda *a: 0)
    monkeypatch.setattr(yvf, "_same_device", lambda *ts: ts[0].device)
    monkeypatch.setattr(yvf, "_training", weakref.WeakSet())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    return stream


def leaf(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).requires_grad_(True)


def off_by_four_bytes(t):
    """A view of t's numbers that starts off 16 bytes (a leaf like t)."""
    flat = torch.zeros(t.numel() + 8, dtype=t.dtype)
    at = next(i for i in range(8) if (flat.data_ptr() + i * t.element_size()) % 16 == 4)
    return flat[at:at + t.numel()].view(t.shape).detach().requires_grad_(True)


# how a leaf reaches the call
WAYS = {
    "itself": lambda w: w,
    "a view": lambda w: w.view(-1).view(w.shape),
    "a cast": lambda w: w.double().float(),
    "a scaled copy": lambda w: (w * 2).view(w.shape),
}


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("which", [0, 1, 3])
def test_a_warm_up_whose_output_lives(captured, way, which):
    """The usual recipe, a warm-up on a side stream and then a captured step, with the warm-up's loss still bound."""
    shared = leaf(4, 4)

    def step():
        ts = [leaf(4, 4) for _ in range(4)]
        ts[which] = WAYS[way](shared)
        return yvf.swiglu(*ts).sum()
    captured[0] = 3
    loss = step()
    loss.backward()  # nothing else lives
    captured[0] = 7
    again = step()
    with pytest.raises(RuntimeError, match="another stream lives"):
        again.backward()
    del loss
    step().backward()


def test_a_leaf_that_is_copied_to_an_aligned_address(captured):
    w = off_by_four_bytes(torch.zeros(4, 4))
    assert w.data_ptr() % 16 != 0 and w.is_leaf
    captured[0] = 3
    kept = yvf.swiglu(torch.zeros(4, 4), w, leaf(4, 4), leaf(4, 4))
    captured[0] = 7
    with pytest.raises(RuntimeError, match="another stream lives"):
        yvf.swiglu(torch.zeros(4, 4), w, leaf(4, 4), leaf(4, 4)).sum().backward()
    del kept


def test_graphs_that_share_no_leaf(captured):
    """Other leaves, the same stream, and an activation that was a view's base and is gone refuse nothing."""
    captured[0] = 3
    base = leaf(2, 2, 4) * 1
    other = yvf.swiglu(base, leaf(4, 4), leaf(4, 4), leaf(4, 4))
    (ctx,) = yvf._training
    assert id(base) not in ctx.leaves and len(ctx.leaves) == 3
    del ctx, base
    captured[0] = 7
    w = leaf(4, 4)
    same = yvf.swiglu(torch.zeros(4, 4), w, leaf(4, 4), leaf(4, 4))
    yvf.swiglu(torch.zeros(4, 4), w, leaf(4, 4), leaf(4, 4)).sum().backward()
    del other, same


def test_calls_of_another_thread(captured):
    """One thread's calls are recorded while another's backward pass looks through them."""
    captured[0] = 7
    stop, w = threading.Event(), [leaf(4, 4) for _ in range(3)]

    def train():
        while not stop.is_set():
            kept = [yvf.swiglu(torch.zeros(4, 4), *w) for _ in range(20)]
            del kept
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    threads = [threading.Thread(target=train) for _ in range(2)]
    try:
        for t in threads:
            t.start()
        mine = yvf.swiglu(torch.zeros(4, 4), *w)
        for _ in range(2000):
            yvf._refuse_other_streams(mine.grad_fn)
    finally:
        stop.set()
        for t in threads:
            t.join()
        sys.setswitchinterval(interval)
