"""Codes at the largest scales of the 8-bit cache's restatement: what they stand for is finite."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv_cache as kv


@pytest.mark.parametrize("byte", range(240, 255))
def test_codes_stand_for_finite_values(byte):
    """Every finite fp32 value of a scale's range: within half a step (2^-4) and below 2^128, as infinity is not."""
    scale = 2.0 ** (byte - 127)
    size = np.linspace(2.0 ** -6, 448, 4001)
    x = np.minimum(size * scale, float(np.finfo(np.float32).max))
    x = np.concatenate([x, -x])
    codes = kv.keep_finite(kv.encode(x / scale), byte)
    got = kv.E4M3[codes] * scale
    assert (np.abs(got) < 2.0 ** 128).all() and (np.abs(got - x) <= 2.0 ** -4 * np.abs(x)).all()
    plain = kv.encode(x / scale)
    np.testing.assert_array_equal(codes[np.abs(kv.E4M3[plain] * scale) < 2.0 ** 128],
                                  plain[np.abs(kv.E4M3[plain] * scale) < 2.0 ** 128])
    assert byte < 247 or (codes != plain).any()
    assert kv.keep_finite(np.array([127, 255], np.uint8), byte).tolist() == [127, 255]
