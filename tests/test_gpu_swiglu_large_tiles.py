"""Training steps whose backward products run in 256 x 256 tiles, each in one piece, as those of large batches do: dh with g
and u read and dg, du and h written (2304 x 1032 x 4100), the gradients of both gate and up weights with rows between them
that belong to neither (4100 is not a multiple of 8), dx, y and the gradient of the down weight (2304 x 4104 x 2050).
Tolerances as in test_gpu_swiglu.py; the 64-bit products run on the GPU."""
import math

import pytest
import torch

from pisceslx_amd import functional as yvf
from test_gpu_swiglu import check, make, step

pytestmark = pytest.mark.gpu


def exact(x, wg, wu, wd, dy, cuda):
    """test_gpu_swiglu.exact, on the GPU."""
    x, wg, wu, wd, dy = (t.to(cuda).double() for t in (x, wg, wu, wd, dy))
    t = lambda a: a.t().contiguous()
    g, u = x @ t(wg), x @ t(wu)
    s = 1 / (1 + torch.exp(-g))
    h, dh = g * s * u, dy @ wd
    du, dg = dh * g * s, dh * u * s * (1 + g * (1 - s))
    ga, ua = x.abs() @ t(wg.abs()), x.abs() @ t(wu.abs())
    ha = s * (g.abs() * ua + u.abs() * ga * (1 + g.abs() * (1 - s)))
    dha, s1 = dy.abs() @ wd.abs(), s * (1 - s)
    dua = dha * (g * s).abs() + dh.abs() * (s + g.abs() * s1) * ga
    dga = dha * u.abs() * s * (1 + g.abs()) + dh.abs() * (s * (1 + g.abs()) * ua + u.abs() * s1 * (2 + g.abs()) * ga)

    def outs(h, dg, du, x, wg, wu, wd, dy):
        return [v.cpu() for v in (h @ t(wd), dg @ wg + du @ wu, t(dg) @ x, t(du) @ x, t(dy) @ h)]
    sizes = [v.abs() for v in (x, wg, wu, wd, dy)]
    return outs(h, dg, du, x, wg, wu, wd, dy), outs(ha, dga, dua, *sizes), outs(h.abs(), dg.abs(), du.abs(), *sizes)


@pytest.mark.parametrize("N,H,F,dtype", [(2304, 1032, 4100, torch.bfloat16), (2304, 4104, 2050, torch.bfloat16),
                                         (2304, 1032, 4100, torch.float32)])
def test_step(cuda, N, H, F, dtype):
    t = make(N, H, F, dtype, seed=2)
    got, again = step(*t, cuda), step(*t, cuda)
    want, size, own = exact(*t, cuda)
    for name, a, c, b, s, o, n in zip(("y", "dx", "dgate", "dup", "ddown"), got, again, want, size, own,
                                      (F + H, 2 * F + H, N + H, N + H, N + H)):
        check(a, b, s, o, dtype, n, f"{name} {N} x {H} x {F}")
        assert torch.equal(a, c), name


def test_one_of_the_gradients(cuda):
    """The up weight's gradient without the gate's, and y of the pass that keeps nothing: the same bits."""
    x, wg, wu, wd, dy = (v.to(cuda) for v in make(2304, 1032, 4100, torch.bfloat16, seed=2))
    full = step(x, wg, wu, wd, dy, cuda)
    w = wu.clone().requires_grad_(True)
    y = yvf.swiglu(x, wg, w, wd)
    y.backward(dy)
    assert torch.equal(w.grad, full[3]) and torch.equal(y.detach(), full[0])
    with torch.no_grad():
        assert torch.equal(yvf.swiglu(x, wg, wu, wd), full[0])
