"""The division that turns rows into codes (csrc/attn_cache_gfx950.h, Divide), step by step in fp32: r = 1 / s, corrected once, q = x r, corrected once.

Let r be the fp32 number nearest to 1 / s, u = 2^-24: s r = 1 + e, |e| <= u.  q is within 2 units of the quotient Q: one rounding in r, one in the product, relative u each, of a Q below twice its unit's power of
two.  The remainder x - s q has 25 bits at most, so that rounding leaves it 2^-25 of itself off.  The last step rounds q + (Q - q)(1 + e) (1 + 2^-25): off from Q by 2 units times (u + 2^-25), 3 units times 2^-24.  That
can round to another number than Q only where Q is as close to the middle of two: with whole numbers 2^23 <= x, s < 2^24 and m odd, |2^24 x - m s| / (2 s) units (Q above 1; 2^25 below), so that |2^24 x - m s| <= 5.  Of
each s there are a handful of such x, which are all found from m = d / s mod 2^24: 29 million, here those of some s (all of them, once: none is off).

The instruction's reciprocal is good to one unit, and after its correction the nearest one (on the device, for each of the 2^23 significands: so it is).  From one unit alone that would follow for all s but those
next to a power of two: 2^24 - 1 and 2^24 - 3 have one x each that would be rounded the other way."""
import numpy as np
import pytest

f32, f64 = np.float32, np.float64


def fma(a, b, c):
    """a b + c of fp32, rounded once: the product is exact in 64 bits, the sum is rounded to odd there."""
    a, b = a.astype(f64) * b.astype(f64), c.astype(f64)
    s = a + b
    t = s - a
    left = (a - (s - t)) + (b - t)
    even = (s.view(np.int64) & 1) == 0
    return np.where((left != 0) & even, np.nextafter(s, np.where(left > 0, np.inf, -np.inf)), s).astype(f32)


def divided(x, s, off):
    """The quotient, and whether the corrected reciprocal is the nearest one, for an instruction that is `off` units off."""
    r = ((f32(1) / s).view(np.int32) + np.int32(off)).view(f32)
    r = fma(fma(-s, r, np.ones_like(s)), r, r)
    q = x * r
    return fma(fma(-s, q, x), r, q), r == f32(1) / s


def inverse(s, bits):
    """1 / s modulo 2^bits, s odd."""
    r = s.copy()
    for _ in range(5):
        r = (r * (2 - s * r)) & ((1 << bits) - 1)
    return r


def hard(s):
    """Pairs (x, s) of 24 bits whose quotient is 5 / (2 s) units or less from the middle of two fp32 numbers."""
    for t in range(3):
        of = s[(s & ((2 << t) - 1)) == 1 << t]
        for d in (-5, -4, -3, -2, -1, 1, 2, 3, 4, 5):
            if d % (1 << t) or not d >> t & 1:
                continue
            for bits in (24, 25):
                low = ((d >> t) * inverse(of >> t, bits - t)) & ((1 << (bits - t)) - 1)
                for i in range(1 << t):
                    m = low + (i << (bits - t)) + ((1 << 24) if bits == 24 else 0)
                    x = m * of - d
                    assert not (x & ((1 << bits) - 1)).any()
                    x >>= bits
                    ok = (m >> 24 == 1) & (x >> 23 == 1)
                    yield x[ok], of[ok]


def check(s):
    count = 0
    for x, of in hard(s):
        count += len(x)
        a, b = x.astype(f32), of.astype(f32)
        # hard they are: their quotient in 64 bits is all but the middle of two numbers of 24 bits
        q = x.astype(f64) / of.astype(f64)
        assert (np.abs(np.abs(q - (a / b).astype(f64)) / np.spacing(a / b).astype(f64) - 0.5) < 2.0 ** -20).all()
        right(a, b)
    return count


def right(x, s):
    for off in (-1, 0, 1):
        got, nearest = divided(x, s, off)
        assert (got == x / s)[nearest].all() and (off or nearest.all())


@pytest.mark.parametrize("first", [0, 1, 2, 4])
def test_quotients_next_to_the_middle_of_two_numbers(first):
    assert check(np.arange((1 << 23) + first, 1 << 24, 4 * 251, dtype=np.int64)) > 5000


def test_significands_of_ones_and_powers_of_two():
    at = np.array([(1 << 24) - 1, (1 << 24) - 2, (1 << 24) - 3, (1 << 23) + 1, (1 << 23) + 2], dtype=np.int64)
    for x, s in hard(at):
        x, s = x.astype(f32), s.astype(f32)
        assert (divided(x, s, 0)[0] == x / s).all()
    x = (np.random.default_rng(0).integers(1 << 23, 1 << 24, 1 << 18)).astype(f32)
    for s in (f32((1 << 24) - 1), f32(1 << 23), f32((1 << 23) + 1)):
        assert (divided(x, np.full_like(x, s), 0)[0] == x / s).all()


def test_any_numbers():
    g = np.random.default_rng(1)
    right(*(g.uniform(0.5, 1, 1 << 20).astype(f32) for _ in range(2)))
