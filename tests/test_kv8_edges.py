"""CPU: the ends of the 8-bit cache's ranges in the float64 restatement."""
import numpy as np
import pytest

from oracle import kv8_ref as R

LARGEST = {"e4m3": 240 * 2.0 ** 120, "int8": 127 * 2.0 ** 121}      # code * 2^e: the next one up is 2^128


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("x", [3.4028234e38, 3.3895314e38, 3.3e38, 3.2e38, 3.1e38, 2.9e38, np.inf])
def test_what_is_kept_of_a_finite_value_is_finite(fmt, x):
    """a value next to fp32's largest is not rounded to 2^128: e4m3 within its half step (2^-4 of the value), int8 within a 127th of the block's largest, as elsewhere"""
    k = np.full((3, 1, 64), x, np.float32)
    k[1], k[2] = -k[1], 2.9e38
    codes, scales = np.zeros((1, 2, 1, 1024), np.uint8), np.zeros((1, 2, 1), np.float32)
    R.append(k, k, codes, scales, fmt, [0, 3], [0], ([0, 1], [0]))
    for got in R.read(codes, scales, fmt, 64, [0, 3], [0], ([0, 1], [0])):
        assert np.isfinite(got.astype(np.float32)).all() and np.abs(got).max() <= LARGEST[fmt]
        if np.isfinite(x):
            assert (np.abs(got - k) <= (2.0 ** -4 * np.abs(k) if fmt == "e4m3" else np.abs(k).max() / 127)).all()
