"""Q as the sum of two e4m3 numbers under a power of two per row: how exact the 8-bit prefill's scores are (CPU)."""
import numpy as np
import pytest

from oracle import cache8


def parts(f):
    hi = cache8.to_e4m3(f)
    return hi, cache8.to_e4m3(f - hi)


def bf16_numbers(lo, hi):
    """Every bf16 number within lo .. hi."""
    bits = np.arange(0x7f80, dtype=np.uint32) << 16
    x = bits.view(np.float32).astype(np.float64)
    return x[(x >= lo) & (x <= hi)]


@pytest.mark.parametrize("top", (225.0, 226.0, 255.0, 256.0, 258.0, 384.0, 446.0, 448.0))
def test_exact_above_and_close_below(top):
    """A row is brought to a largest magnitude of 224 (not included) to 448.  From 1/4 on, 2^-9.8 of the largest at most, the sum is
    exact; below it is off by half of e4m3's least step, 2^-10, which is less than 2^-17.8 of the largest."""
    assert 224 < top <= 448
    f = bf16_numbers(0.25, top)
    hi, lo = parts(f)
    assert np.array_equal(hi + lo, f) and 0.25 / top <= 2.0 ** -9.8
    f = bf16_numbers(2.0 ** -130, 0.25)
    hi, lo = parts(f)
    off = np.abs(hi + lo - f)
    assert off.max() == 2.0 ** -10 and 2.0 ** -10 / top < 2.0 ** -17.8
    hi, lo = parts(-f)
    assert np.array_equal(np.abs(hi + lo + f), off)


def test_the_bounds_are_tight():
    """The number in front of 1/4 is not exact, and an error reaches more than 2^-18 of a largest magnitude of 225."""
    x = 0.25 - 2.0 ** -10
    hi, lo = parts(np.array([x]))
    assert hi[0] + lo[0] == 0.25 and x / 225 > 2.0 ** -11 and 2.0 ** -10 / 225 > 2.0 ** -18
