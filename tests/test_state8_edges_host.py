"""The edges of the 8-bit state's code in the oracle, without a GPU."""
import numpy as np
import pytest

from oracle import state8 as S8

LARGEST = np.finfo(np.float32).max


@pytest.mark.parametrize('top', [LARGEST, np.float32(1.9375 * 2.0**127), np.float32(1.75 * 2.0**127)])
def test_what_is_finite_stays_finite(top):
    x = np.random.default_rng(0).random((2, 256)).astype(np.float32) * np.float32(1e38)
    x[0, 9] = x[1, 255] = top
    dithers = (S8.HALF, np.full((2, 256), (1 << 20) - 1))
    for sign in (1, -1):
        once = S8.decode_avg(*S8.encode_avg(sign * x))
        assert np.all(np.isfinite(once)) and np.all(np.abs(once / (sign * x) - 1) <= 2.0**-4)
        np.testing.assert_array_equal(S8.decode_avg(*S8.encode_avg(once)), once)
    for r in dithers:
        once = S8.decode_sq(*S8.encode_sq(x, r))
        assert np.all(np.isfinite(once)) and np.all(np.abs(once / x - 1) <= 2.0**-3)
        np.testing.assert_array_equal(S8.decode_sq(*S8.encode_sq(once, S8.HALF)), once)


def test_a_sign_of_exp_avg_sq_is_dropped():
    x = np.random.default_rng(0).random((1, 256)).astype(np.float32)
    x[0, ::5] *= -1
    x[0, 7] = -0.0
    codes, e = S8.encode_sq(x, S8.HALF)
    want, we = S8.encode_sq(np.abs(x), S8.HALF)
    assert np.array_equal(codes, want) and np.array_equal(e, we) and codes[0, 7] == 0
