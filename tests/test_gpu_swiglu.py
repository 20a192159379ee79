"""The gated feed-forward block and its gradients against a 64-bit evaluation of the formulas.

Tolerances. bf16, u = 2^-9 the rms-free half step of a rounding (eps / 2 = 2^-8 relative at most, uniformly
spread: 2^-8 / sqrt(3) rms): y has h's and its own rounding, dx those of dg and du and its own, dWg, dWu, dWd
that of one operand and its own. Each is a random sum whose terms are off by at most 2^-8 relative and by
2^-8 / sqrt(3) = 2.26e-3 rms at the very most (a mantissa of 1; on average over mantissas 0.72 of that), so the
2-norm of the error is under sqrt(2) 2.26e-3 = 3.2e-3 of the 2-norm of a sum with terms of random signs; the
same holds for a single product (N = 1, F = 1), where both roundings may add: 2 * 2^-8 = 7.9e-3. A single element
is off by at most 2^-8 of itself plus 2^-8 of the sum of its terms' sizes: compared against that, computed in 64
bits. fp32: three bf16 terms leave 2^-24 relative of an operand, and the sum of n products in fp32 at most
n 2^-24 of the sum of sizes, sqrt(n) of that typically; 6 sqrt(n) + 40 half steps of 2^-24 are allowed on the
sum of sizes (40: expf, the products of the activation and its derivative, each within a few half steps).
"""
import math

import pytest
import torch

from pisceslx_amd import functional as yvf

pytestmark = pytest.mark.gpu


def make(N, H, F, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    return ((r(N, H) * scale).to(dtype), (r(F, H) / math.sqrt(H)).to(dtype), (r(F, H) / math.sqrt(H)).to(dtype),
            (r(H, F) / math.sqrt(F)).to(dtype), r(N, H).to(dtype))


def exact(x, wg, wu, wd, dy):
    """Outputs and the sums of the sizes of their terms, in 64 bits on the CPU."""
    x, wg, wu, wd, dy = (t.double().cpu() for t in (x, wg, wu, wd, dy))
    g, u = x @ wg.t(), x @ wu.t()
    s = 1 / (1 + torch.exp(-g))
    h = g * s * u
    dh = dy @ wd
    du, dg = dh * g * s, dh * u * s * (1 + g * (1 - s))
    out = (h @ wd.t(), dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h)
    # sizes: what an operand's error is measured against includes the error of the sums that made it
    ga, ua = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t()
    ha = s * (g.abs() * ua + u.abs() * ga * (1 + g.abs() * (1 - s)))
    dha = dy.abs() @ wd.abs()
    s1 = s * (1 - s)
    dua = dha * (g * s).abs() + dh.abs() * (s + g.abs() * s1) * ga
    dga = dha * u.abs() * s * (1 + g.abs()) + dh.abs() * (s * (1 + g.abs()) * ua + u.abs() * s1 * (2 + g.abs()) * ga)
    size = (ha @ wd.abs().t(), dga @ wg.abs() + dua @ wu.abs(), dga.t() @ x.abs(), dua.t() @ x.abs(),
            dy.abs().t() @ ha)
    own = (h.abs() @ wd.abs().t(), dg.abs() @ wg.abs() + du.abs() @ wu.abs(), dg.abs().t() @ x.abs(),
           du.abs().t() @ x.abs(), dy.abs().t() @ h.abs())
    return out, size, own


def check(got, want, size, own, dtype, n, name):
    got = got.double().cpu()
    fp32 = (6 * math.sqrt(n) + 40) * 2.0 ** -24 * size
    bound = fp32 + 1e-30 if dtype == torch.float32 else 2.0 ** -8 * (want.abs() + own * 1.01) + fp32
    off = (got - want).abs()
    worst = float((off / bound.clamp(min=1e-300)).max()) if off.numel() else 0.0
    rel = float(off.norm() / want.norm().clamp(min=1e-300))
    print(f"{name}: worst / bound {worst:.3f}, rel {rel:.2e}", flush=True)
    assert torch.isfinite(got).all() and worst <= 1.0, name
    if dtype == torch.bfloat16:
        assert rel <= (3.2e-3 if min(got.shape) > 8 and n > 8 else 7.9e-3), name


def step(x, wg, wu, wd, dy, cuda):
    leaves = [t.detach().to(cuda).requires_grad_(True) for t in (x, wg, wu, wd)]
    y = yvf.swiglu(*leaves)
    return (y.detach(), *torch.autograd.grad(y, leaves, dy.to(cuda)))


SIZES = [(1, 1, 1), (1, 8, 8), (2, 64, 64), (3, 7, 5), (5, 128, 96), (16, 256, 320), (17, 100, 130), (33, 72, 264),
         (64, 512, 128), (65, 63, 129), (130, 257, 255), (200, 384, 1000), (300, 1000, 272),
         (100, 100, 204), (1000, 36, 68), (66, 1028, 772), (90, 2048, 1536)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("N,H,F", SIZES)
def test_step(cuda, N, H, F, dtype):
    t = make(N, H, F, dtype, seed=N + H + F)
    got = step(*t, cuda)
    want, size, own = exact(*t)
    for name, a, b, s, o, n in zip(("y", "dx", "dgate", "dup", "ddown"), got, want, size, own,
                                   (F + H, 2 * F + H, N + H, N + H, N + H)):
        assert a.shape == b.shape and a.dtype == dtype
        check(a, b, s, o, dtype, n, f"{name} {N} x {H} x {F}")
    # without gradients the same bits
    with torch.no_grad():
        assert torch.equal(yvf.swiglu(*(v.to(cuda) for v in t[:4])), got[0])


# tiles of 256 and 128, with full and partial ends, and the same bits twice
@pytest.mark.parametrize("N,H,F,dtype", [(2050, 1032, 3080, torch.bfloat16), (777, 2056, 1544, torch.bfloat16),
                                         (1500, 1024, 2816, torch.float32), (515, 1001, 2003, torch.float32),
                                         (515, 1001, 2003, torch.bfloat16), (1020, 516, 2052, torch.float32),
                                         (1030, 516, 2052, torch.float32)])
def test_step_large(cuda, N, H, F, dtype):
    t = make(N, H, F, dtype, seed=1)
    got, again = step(*t, cuda), step(*t, cuda)
    want, size, own = exact(*t)
    for name, a, c, b, s, o, n in zip(("y", "dx", "dgate", "dup", "ddown"), got, again, want, size, own,
                                      (F + H, 2 * F + H, N + H, N + H, N + H)):
        check(a, b, s, o, dtype, n, f"{name} {N} x {H} x {F}")
        assert torch.equal(a, c), name


def test_differences(cuda):
    """Gradients against central differences of the fp32 forward pass: for a direction v of an input, d/dt of
    sum(y dy) at step 2^-5 is off by t²/6 of a third derivative (under 5e-3 here: the activation's is below 1 and
    v has unit size per row) and by the forward's rounding over the step."""
    x, wg, wu, wd, dy = make(40, 48, 56, torch.float32, seed=5)
    got = step(x, wg, wu, wd, dy, cuda)
    t = 2.0 ** -5
    g = torch.Generator().manual_seed(9)
    for i, grad in enumerate(got[1:]):
        ins = [x, wg, wu, wd]
        v = torch.randn(ins[i].shape, generator=g)
        v /= v.norm()
        f = []
        for s in (t, -t):
            a = list(ins)
            a[i] = a[i] + s * v
            f.append((yvf.swiglu(*(q.to(cuda) for q in a)).double().cpu() * dy.double()).sum())
        diff = float((f[0] - f[1]) / (2 * t))
        want = float((grad.double().cpu() * v.double()).sum())
        assert abs(diff - want) <= 5e-3 * float(grad.double().norm()), (i, diff, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_no_rows(cuda, dtype):
    t = make(0, 24, 40, dtype)
    got = step(*t, cuda)
    assert got[0].shape == (0, 24) and got[1].shape == (0, 24)
    for a, b in zip(got[2:], t[1:4]):
        assert a.shape == b.shape and int((a != 0).sum()) == 0


@pytest.mark.parametrize("which", range(1, 15))
def test_some_gradients(cuda, which):
    """Only the inputs that need a gradient get one, the same bits as with all of them."""
    t = make(70, 40, 48, torch.bfloat16, seed=3)
    full = step(*t, cuda)
    leaves = [v.to(cuda).requires_grad_(bool(which >> i & 1)) for i, v in enumerate(t[:4])]
    yvf.swiglu(*leaves).backward(t[4].to(cuda))
    for i, v in enumerate(leaves):
        if which >> i & 1:
            assert torch.equal(v.grad, full[1 + i])
        else:
            assert v.grad is None


def test_shapes_strides_and_broadcast_gradients(cuda):
    """Leading dimensions, tensors that start off 16 bytes, gradients that a sum's backward expands, and one
    weight used twice."""
    x, wg, wu, wd, dy = (t.to(cuda) for t in make(30, 24, 40, torch.bfloat16, seed=4))
    want = yvf.swiglu(x, wg, wu, wd)
    flat = torch.zeros(3 + x.numel() + wg.numel(), dtype=x.dtype, device=cuda)
    xo, wo = flat[3:3 + x.numel()].view_as(x), flat[3 + x.numel():].view_as(wg)
    xo.copy_(x), wo.copy_(wg)
    assert torch.equal(yvf.swiglu(xo.view(5, 6, 24), wo, wu, wd).view(30, 24), want)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    yvf.swiglu(*leaves).sum().backward()
    ones = step(*(t.detach() for t in leaves), torch.ones_like(x), cuda)
    for a, b in zip(leaves, ones[1:]):
        assert torch.equal(a.grad, b)
    a = wg.clone().requires_grad_(True)
    yvf.swiglu(x, a, a, wd).backward(dy)
    both = step(x, wg, wg.clone(), wd, dy, cuda)
    assert torch.equal(a.grad, both[2] + both[3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("N", [3, 100])
def test_rows_that_are_no_numbers(cuda, dtype, N):
    """An infinity or NaN stays in its row of y and dx."""
    x, wg, wu, wd, dy = make(N, 40, 72, dtype, seed=6)
    clean = step(x, wg, wu, wd, dy, cuda)
    x2 = x.clone()
    x2[1, 3] = math.nan
    x2[2, 5] = math.inf
    got = step(x2, wg, wu, wd, dy, cuda)
    keep = torch.ones(N, dtype=torch.bool)
    keep[1:3] = False
    for k in (0, 1):
        assert torch.equal(got[k].cpu()[keep], clean[k].cpu()[keep])
        assert not torch.isfinite(got[k].cpu()[~keep]).any()


def test_large_and_small_gates(cuda):
    """Gates far from zero: exp overflows and underflows, the activation and its derivative stay right."""
    x, wg, wu, wd, dy = make(40, 64, 64, torch.float32, seed=7)
    wg = wg * 200
    got = step(x, wg, wu, wd, dy, cuda)
    want, size, own = exact(x, wg, wu, wd, dy)
    for name, a, b, s, o in zip(("y", "dx", "dgate", "dup", "ddown"), got, want, size, own):
        check(a, b, s, o, torch.float32, 256, name)


def test_captured(cuda):
    """A captured step replays on new inputs, with eager work between the replays."""
    x, wg, wu, wd, dy = (t.to(cuda) for t in make(150, 136, 264, torch.bfloat16, seed=8))
    ins = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(yvf.swiglu(*ins), ins, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = yvf.swiglu(*ins)
        grads = torch.autograd.grad(y, ins, dy)
    for k in range(4):
        new = make(150, 136, 264, torch.bfloat16, seed=20 + k)
        with torch.no_grad():
            for a, b in zip(ins, new[:4]):
                a.copy_(b)
            dy.copy_(new[4])
        graph.replay()
        torch.cuda.synchronize()
        want = step(*new, cuda)
        for a, b in zip((y.detach(), *grads), want):
            assert torch.equal(a, b)


def test_on_another_stream(cuda):
    t = [v.to(cuda) for v in make(100, 64, 96, torch.bfloat16, seed=10)]
    want = step(*t, cuda)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = step(*t, cuda)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N,H,F,dtype", [(2050, 520, 3080, torch.bfloat16), (700, 1000, 1030, torch.bfloat16),
                                         (90, 2048, 1536, torch.bfloat16), (1500, 512, 2050, torch.float32)])
def test_without_gradients_the_same_bits(cuda, N, H, F, dtype):
    """The forward pass that keeps nothing, in tiles of each size and split: the bits of the one that keeps g and u."""
    x, wg, wu, wd, _ = (t.to(cuda) for t in make(N, H, F, dtype, seed=3))
    kept = yvf.swiglu(x.requires_grad_(True), wg, wu, wd).detach()
    with torch.no_grad():
        assert torch.equal(yvf.swiglu(x, wg, wu, wd), kept)


@pytest.mark.parametrize("N", [16, 40, 4000])
def test_activation_by_itself(cuda, N):
    """y = silu(g): x = (g, 1), gate (1, 0), up (0, 1), down 1, whose products are exact. The activation's quotient is
    within six half steps and its product one: 7 x 2^-24 relative. Far gates give g and 0."""
    g = torch.cat([torch.linspace(-60, 90, N - 4), torch.tensor([1000.0, 3e38, -1000.0, 0.0])])
    x = torch.stack([g, torch.ones(N)], 1)
    wd = torch.tensor([[1.0], [0.0]])
    args = [t.to(cuda) for t in (x, torch.tensor([[1.0, 0.0]]), torch.tensor([[0.0, 1.0]]), wd)]
    y = yvf.swiglu(*args).cpu().double()
    want = g.double() / (1 + torch.exp(-g.double()))
    worst = float(((y[:, 0] - want).abs() / (7 * 2.0 ** -24 * want.abs() + 1e-35)).max())
    print(f"silu, {N} rows: worst / bound {worst:.3f}", flush=True)
    assert worst <= 1 and (y[:, 1] == 0).all()
