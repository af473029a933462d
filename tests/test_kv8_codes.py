"""The coding of the 8-bit cache without a division (csrc/sf_kv8.hip, Coder), restated in float32: over every pair of
bf16 significands and every exponent that gives a code, it is rint(127 x / top) of exact arithmetic, ties to even."""
import numpy as np


def _coder(x, top):
    one = np.float32(1)
    unit = np.where(top < 2.0 ** -60, np.float32(2.0 ** 66), np.where(top > 2.0 ** 60, np.float32(2.0 ** -60), one))
    unit = unit.astype(np.float32)
    c = np.float32(127) / (top * unit)
    y = x * unit * c
    t = y * np.float32(65)
    return np.rint(t - (t - y)).astype(np.int64)


def test_every_pair_of_significands():
    a, b = np.meshgrid(np.arange(128, 256), np.arange(128, 256), indexing="ij")
    for shift in range(12):  # x = a 2^-shift against top = b: 127 a / (b 2^shift)
        keep = a <= b * 2 ** shift
        num, den = 127 * a[keep].astype(np.int64), b[keep].astype(np.int64) << shift
        q, r = num // den, num % den
        want = q + ((2 * r > den) | ((2 * r == den) & (q % 2 == 1)))
        for e in (0, -7, 50, 70, -70, -110, 115):
            x = np.ldexp(a[keep].astype(np.float32), e - shift).astype(np.float32)
            top = np.ldexp(b[keep].astype(np.float32), e).astype(np.float32)
            assert np.array_equal(_coder(x, top), want), (shift, e)
            assert np.array_equal(_coder(-x, top), -want), (shift, e)


def test_subnormal_numbers():
    """bf16 below 2^-126 are multiples of 2^-133."""
    a, b = np.meshgrid(np.arange(0, 128), np.arange(1, 128), indexing="ij")
    keep = a <= b
    num, den = 127 * a[keep].astype(np.int64), b[keep].astype(np.int64)
    q, r = num // den, num % den
    want = q + ((2 * r > den) | ((2 * r == den) & (q % 2 == 1)))
    x, top = (np.ldexp(t[keep].astype(np.float64), -133).astype(np.float32) for t in (a, b))
    assert np.array_equal(_coder(x, top), want)
