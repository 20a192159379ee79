"""The quotient behind the 8-bit codes: q = a r, then q + r (a - q s) with r = 1 / s, each rounded to fp32 once, gives the
codes of the rounded division.

Both are rounded from within 2^-22 of an fp32 step of a / s, so they differ only where a / s lies as near the middle of two
fp32 numbers, and a code differs only if one of these two is a border between codes, t / 16 times a power of two, t from 16
to 31. With a and s as 24-bit whole numbers that takes 16 a - t s = j, a whole number, with j / (16 s) half an fp32 step of
the quotient, 2^-24 or 2^-25 of a power of two: j = 16 s 2^-24 (or half of that), at most 16 in size and within a few millionths
of a whole number, so s lies within a few steps of a multiple of 2^20. All such quotients are tried, with room: s within 24
steps, |j| up to 40. In numpy: products of two fp32 numbers are exact in 64 bits, a - q s is too, and the last sum is rounded
to odd before it is rounded to fp32."""
from fractions import Fraction as F

import numpy as np
import pytest
import torch


def fma_last(x, y, z):
    """x y + z of fp32 numbers, rounded once."""
    p, z = x.astype(np.float64) * y.astype(np.float64), z.astype(np.float64)
    s = p + z
    b = s - p
    lost = (p - (s - b)) + (z - b)  # s + lost = p + z exactly
    bits = s.view(np.int64)
    # rounded to odd: where something was lost from an even s, its neighbour on that side
    step = np.where((lost > 0) == (s > 0), 1, -1)
    odd = np.where((lost != 0) & (bits & 1 == 0), bits + step, bits)
    return odd.view(np.float64).astype(np.float32)


def quotient(a, s):
    r = np.float32(1) / s
    q = a * r
    rest = (a.astype(np.float64) - q.astype(np.float64) * s.astype(np.float64)).astype(np.float32)
    return fma_last(rest, r, q)


def codes(v):
    return torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8)


def test_all_quotients_beside_a_border():
    multiples = np.arange(8, 17, dtype=np.int64)[:, None] << 20
    s = (multiples + np.arange(-24, 25)).ravel()
    s = s[(s >= 1 << 23) & (s < 1 << 24)][:, None, None]
    t, j = np.arange(16, 32)[None, :, None], np.arange(-40, 41)[None, None, :]
    n = t * s + j
    s = np.broadcast_to(s, n.shape)
    a = n >> 4
    fits = (n & 15 == 0) & ((a < 1 << 24) | (a & 1 == 0))  # of 24 bits
    a, s = a[fits].astype(np.float32), s[fits].astype(np.float32)
    assert len(a) > 20000
    ours, divided = quotient(a, s), a / s
    print(f"{len(a)} quotients, {int((ours != divided).sum())} not the rounded one")
    for k in (0, -6, -8, -9, -10):  # normal codes, and subnormal ones, whose borders are some of these
        assert torch.equal(codes(np.ldexp(ours, k)), codes(np.ldexp(divided, k)))


@pytest.mark.parametrize("seed", range(4))
def test_quotients_at_random(seed):
    g = np.random.default_rng(seed)
    s = g.integers(1 << 23, 1 << 24, 1 << 20).astype(np.float32)
    a = np.where(g.random(1 << 20) < 0.5, np.rint(s.astype(np.float64) * g.integers(16, 32, 1 << 20) / 16
                                                  + g.integers(-3, 4, 1 << 20)), g.integers(1 << 23, 1 << 25, 1 << 20))
    a = a.astype(np.float32)
    assert torch.equal(codes(quotient(a, s)), codes(a / s))


def test_the_last_sum():
    """fma_last against whole numbers."""
    g = np.random.default_rng(9)
    x, y, z = (g.integers(1 << 23, 1 << 24, 2000).astype(np.float32) for _ in range(3))
    x, z = np.ldexp(x, -24) * np.where(g.random(2000) < 0.5, -1, 1).astype(np.float32), z
    x, y = np.ldexp(x, -23), np.ldexp(y, -23)
    for a, b, c, got in zip(x, y, z, fma_last(x, y, z)):
        want = F(float(a)) * F(float(b)) + F(float(c))
        near = [np.nextafter(got, np.float32(d)) for d in (-np.inf, np.inf)]
        off = abs(F(float(got)) - want)
        assert all(off <= abs(F(float(v)) - want) for v in near)
