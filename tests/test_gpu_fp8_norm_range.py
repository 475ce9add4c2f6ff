"""The norm into 8 bits over rows whose root mean square, or its inverse, lies past what fp32 holds as a normal number:
to the bit."""

from __future__ import annotations

import pytest
import torch

from fp4_helpers import activations
from oracle import fp4 as ora
from test_gpu_fp4_quant import _same_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [32, 512, 4128, 16384])
@pytest.mark.parametrize("power", [-132, -130, -128, -127, -60, -50, -49, 48, 50, 60, 120, 123])
def test_powers(pkg, power, k):
    """Rows of 2^power and their like, down to bf16's subnormals and up to its largest values, with no eps."""
    x = activations(6, k, k).clamp(-12, 12)
    x = (x.double() * 2.0 ** power).to(torch.bfloat16)
    x[2] = 0.0
    x[2, k // 2] = 2.0 ** power  # one value of a row
    x[4] = 2.0 ** power
    w = activations(1, k, 9)[0]
    _, rows = pkg.ops.add_rmsnorm_fp8(x.cuda(), None, w.cuda(), 0.0)
    _same_rows(rows, *ora.quantize_rows(ora.add_norm(x, None, w, 0.0)[1]))
    assert not bool(torch.isnan(rows.codes.float()).any())


def test_the_smallest_and_the_largest_value(pkg):
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    x[0, 5] = 2.0 ** -133
    x[1] = torch.finfo(torch.bfloat16).max
    x[2], x[2, 0] = 2.0 ** -133, -(2.0 ** -133)
    w = torch.ones(64, dtype=torch.bfloat16)
    for eps in (0.0, 1e-300, 1e-5):
        _, rows = pkg.ops.add_rmsnorm_fp8(x.cuda(), None, w.cuda(), eps)
        _same_rows(rows, *ora.quantize_rows(ora.add_norm(x, None, w, eps)[1]))


@pytest.mark.parametrize("eps", [1e-80, 1e-30, 1e30])
def test_eps(pkg, eps):
    """An eps that puts the root past the range by itself."""
    x = activations(5, 544, 3)
    x[1] = 0
    w = activations(1, 544, 9)[0]
    for scale in (1e-38, 1.0, 1e36):
        scaled = (x.double().clamp(-12, 12) * scale).to(torch.bfloat16)
        _, rows = pkg.ops.add_rmsnorm_fp8(scaled.cuda(), None, w.cuda(), eps)
        _same_rows(rows, *ora.quantize_rows(ora.add_norm(scaled, None, w, eps)[1]))
