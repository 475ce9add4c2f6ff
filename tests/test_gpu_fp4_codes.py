"""Every weight code with every scale through the products, exactly: one such weight among zeros times one is the weight
itself, rounded to bf16 (infinite from 2^128 on, and NaN with the scale 255)."""

from __future__ import annotations

import pytest
import torch

from fp4_choice import choice
from fp4_helpers import E8, F8, weight
from oracle import fp4 as ora

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,tile", [(1, 0), (20, 0), (260, 32), (300, 64), (1500, 128)])
def test_every_weight(pkg, m, tile, rows):
    n, k = 16 * 256, 64
    if tile:
        assert choice(pkg, m, n, k, rows, False)[0] >= 32
    code = torch.zeros(n, k, dtype=torch.int64)
    at = torch.arange(n)
    place = at * 7 % k  # each row's own
    code[at, place] = at % 16
    byte = torch.full((n, k // 32), 127)
    byte[at, place // 32] = at // 16
    x = torch.ones(m, k, dtype=torch.bfloat16, device="cuda")
    held = pkg.ops.Fp8Rows(x.to(F8), torch.full((m, k // 32), 127, dtype=torch.uint8, device="cuda").view(E8))
    w = weight(pkg, code, byte)
    y = pkg.ops.w4a8_linear(held, w) if rows else pkg.ops.w4a16_linear(x, w)
    want = ora.weight_values(code, byte)[at, place].to(torch.bfloat16)
    want[byte[at, place // 32] == 255] = float("nan")
    assert torch.equal(torch.nan_to_num(y.float().cpu(), nan=7.0, posinf=8.0, neginf=9.0),
                       torch.nan_to_num(want.float(), nan=7.0, posinf=8.0, neginf=9.0).expand(m, n))
