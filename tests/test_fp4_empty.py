"""4-bit weights of no rows or no columns through what needs no kernel, without a GPU."""

from __future__ import annotations

import pytest
import torch

from fp4_helpers import E8


@pytest.mark.parametrize("n,k", [(0, 128), (0, 544), (16, 0), (0, 0)])
def test_unpacking_and_values(pkg, n, k):
    ops = pkg.ops
    w = ops.Fp4Weight(torch.zeros(-(-n // 16), -(-k // 128), 1024, dtype=torch.uint8),
                      torch.zeros(-(-n // 16), -(-k // 512), 256, dtype=torch.uint8), n, k)
    codes, scales = ops.unpack_fp4(w)
    assert codes.shape == (n, k // 2) and scales.shape == (n, k // 32) and scales.dtype == E8
    assert ops.dequantize_fp4(codes, scales).shape == (n, k)


@pytest.mark.parametrize("mode", ["w4a16", "w4a8"])
def test_modules(pkg, mode):
    assert pkg.Fp4Linear(64, 0, mode).dequantized().shape == (0, 64)
    assert pkg.Fp4Linear(0, 16, mode).dequantized().shape == (16, 0)
