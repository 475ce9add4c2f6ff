"""The 4-bit oracle against brute force, without a GPU."""

from __future__ import annotations

import torch

from oracle import fp4 as ora


def test_scales_are_the_smallest_that_hold_the_group():
    g = torch.Generator().manual_seed(0)
    v = torch.randn(200, 32, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-120, 120, (200, 1), generator=g))
    for top in (6.0, 448.0):
        byte = ora.scale_bytes(v, top)
        s = torch.exp2(byte.double() - 127)
        amax = v.abs().amax(-1)
        assert bool((amax <= top * s).all()) and bool(((amax > top * s / 2) | (byte == 1)).all())
    assert ora.scale_bytes(torch.zeros(1, 32, dtype=torch.float64), 6.0).item() == 1
    assert ora.scale_bytes(torch.full((1, 32), 6.0, dtype=torch.float64), 6.0).item() == 127
    assert ora.scale_bytes(torch.full((1, 32), 6.0001, dtype=torch.float64), 6.0).item() == 128


def test_weight_codes_are_the_nearest():
    v = torch.linspace(-6, 6, 32 * 25).view(25, 32)
    v[:, 0] = 6.0  # scale 1
    code, byte = ora.quantize_weight(v)
    assert bool((byte == 127).all())
    values = ora.weight_values(code, byte)
    every = torch.cat([ora.FP4, -ora.FP4])
    best = (v.double()[..., None] - every).abs().amin(-1)
    assert torch.equal((values - v.double()).abs(), best)
    ties, _ = ora.quantize_weight(torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4]))
    assert ties[0, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 7]


def test_row_codes_are_torchs():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(50, 64, generator=g)
    v, byte = ora.quantize_rows(x)
    scaled = (x.unflatten(-1, (-1, 32)) * torch.exp2(127 - byte.float())[..., None]).flatten(-2)
    assert torch.equal(v.float(), scaled.to(torch.float8_e4m3fn).float())


def test_products_of_small_numbers():
    code, byte = torch.tensor([[2, 10, 7, 0] * 8]), torch.tensor([[128]])  # 2, -2, 12, 0
    y, s = ora.product(torch.ones(1, 32), ora.weight_values(code, byte))
    assert y.item() == 8 * 12 and s.item() == 8 * 16
