"""The few-token layer's experts in 64 bits with h as it is, and the tolerance of a kernel that keeps 16 bits of h."""
import torch

U32, BF16 = 2.0 ** -24, torch.bfloat16


def dense(ex, e):
    """((Wg, Wu, Wd), what their 32-bit sums are made of) in 64 bits: |W|, for int4 the sums of up to 15 s |x| with
    8 s |x| taken off again."""
    ws = [w.double() for w in ex.dequantize(e, torch.float64)]
    if ex.s_gate is None or ex.s_gate.dim() != 3 or ex.s_gate.dtype != BF16:
        return ws, [w.abs() for w in ws]
    return ws, [23 * s[e].double().abs().repeat_interleave(128, -1) for s in (ex.s_gate, ex.s_up, ex.s_down)]


def exact(x, w, idx, experts, E, mix, skip, h_of=lambda h: h):
    """(out, shared, tolerances without the outputs' rounding). experts(e): as dense gives. h_of: a model of how h is
    kept; the tolerance is that of two bf16 terms, whatever it is.

    * 32-bit sums of n products: 2 sqrt(n) half-steps of the sum of their magnitudes. Those of gate and up reach h
      with 1.1 for silu's steepest place and 8 half-steps for its own arithmetic.
    * h in two bf16 terms: what the first leaves is at most 2^-8 |h|, and the second's rounding at most 2^-8
      of that: 2^-16 |h|.
    * the errors of one row's h are independent, so that Wd adds up their squares: four times the root.
    * the weighted sum: F is cut into F / 64 parts at most, so slots F / 64 terms, and 2 sqrt(their number)
      half-steps of the magnitudes."""
    x = x.double()
    N, H = x.shape
    out = torch.zeros(N, H, dtype=torch.float64, device=x.device)
    tol, shared, stol = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(out)

    def expert(e, t, scale, into, tinto, slots):
        (g, u, d), (ga, ua, da) = experts(e)
        xs = x[t]
        gs, us = xs @ g.t(), xs @ u.t()
        n = 2 * H ** 0.5 * U32
        act = torch.nn.functional.silu(gs)
        h = act * us
        err = 1.1 * n * (xs.abs() @ ga.t()) * us.abs() + act.abs() * n * (xs.abs() @ ua.t()) + 8 * U32 * h.abs()
        err = err + 2.0 ** -16 * h.abs()
        F = h.shape[1]
        sums = 2 * (F ** 0.5 + (slots * F / 64) ** 0.5) * U32
        s = scale.double()[:, None]
        into.index_add_(0, t, s * (h_of(h) @ d.t()))
        tinto.index_add_(0, t, s.abs() * (4 * (err.square() @ d.square().t()).sqrt() + sums * (h.abs() @ da.t())))

    for e in range(E):
        t, j = torch.nonzero(idx == e, as_tuple=True)
        if t.numel():
            expert(e, t, w[t, j], out, tol, idx.shape[1])
    S = 0 if mix is None else mix.numel()
    every = torch.arange(N, device=x.device)
    for s in range(S):
        expert(E + s, every, mix[s].expand(N), shared, stol, S)
    out, tol = out + shared, tol + stol
    if skip is not None:
        out = out + 0.1 * skip.double()
    tol = tol + 4 * U32 * (out.abs() + (0 if skip is None else skip.double().abs()))
    return out, shared, tol + 1e-30, stol + 4 * U32 * shared.abs() + 1e-30


def two_terms(h, sign=1.0):
    hi = h.float().to(BF16).double()
    return hi + sign * (h - hi).float().to(BF16).double()


def excess(got, ref, tol):
    """Largest error in units of the tolerance (of the outputs' type: half a step, 2^-8 relative, on top)."""
    return float(((got.double() - ref).abs() / (tol + 1.01 * 2.0 ** -8 * (ref.abs() + tol))).max())


def rounding_ratio(got, ref):
    """Norm of the error against that of rounding the exact outputs once. An h of 16 bits moves a number by some
    2^-17 of itself before it is rounded, by far less than a step, so the ratio is 1 within a few per
    cent; one bf16 term adds a second error of the rounding's size: 1.4."""
    err = (got.double() - ref).norm()
    return float(err / (ref.float().to(BF16).double() - ref).norm())
