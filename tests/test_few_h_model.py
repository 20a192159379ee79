"""On the CPU: the tolerance of tests/few_h_reference.py passes h in two bf16 terms and tells every mistake in the
second term."""
import pytest
import torch

from few_h_reference import BF16, exact, excess, rounding_ratio, two_terms


def one_term(h):
    return h.float().to(BF16).double()


MISTAKES = {
    "dropped": one_term,
    "subtracted": lambda h: two_terms(h, -1.0),
    "doubled": lambda h: two_terms(h, 2.0),
    "of the row before": lambda h: one_term(h) + (two_terms(h) - one_term(h)).roll(1, 0),
    "of the column before": lambda h: one_term(h) + (two_terms(h) - one_term(h)).roll(1, 1),
}


def problem(N, H, E, F, k, S):
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    ws = [[r(F, H) * H ** -0.5, r(F, H) * H ** -0.5, r(H, F) * F ** -0.5] for _ in range(E + S)]
    x, skip = r(N, H).to(BF16), r(N, H).to(BF16)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(N)])
    w = torch.softmax(r(N, k), 1).float()
    mix = torch.softmax(r(S), 0).float() if S else None
    return (x, w, idx, lambda e: (ws[e], [m.abs() for m in ws[e]]), E, mix, skip if S else None)


@pytest.mark.parametrize("N,H,E,F,k,S", [(1, 256, 4, 256, 2, 1), (2, 640, 5, 384, 3, 2), (16, 256, 3, 1280, 2, 1),
                                         (13, 1024, 12, 768, 5, 0)])
def test_the_second_term_counts(N, H, E, F, k, S):
    args = problem(N, H, E, F, k, S)
    ref, sref, tol, stol = exact(*args)
    out, shared, _, _ = exact(*args, h_of=two_terms)
    good = [excess(out.to(BF16), ref, tol), rounding_ratio(out.to(BF16), ref)]
    assert good[0] <= 1.0 and good[1] <= 1.1, good
    assert not S or excess(shared.to(BF16), sref, stol) <= 1.0
    for name, h_of in MISTAKES.items():
        if N == 1 and "row" in name:
            continue
        out, _, _, _ = exact(*args, h_of=h_of)
        bad = [excess(out.to(BF16), ref, tol), rounding_ratio(out.to(BF16), ref)]
        print(f"{N} {H} {F} {name}: {bad[0]:.1f} of the tolerance, ratio {bad[1]:.2f}; right: {good[0]:.2f}, {good[1]:.3f}")
        assert bad[0] > 1.5 and bad[1] > 1.1, (name, bad)
