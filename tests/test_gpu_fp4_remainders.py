"""Every tile kernel of the 4-bit products over every remainder of K in its pipeline: 1 to 12 steps of 128 and some more,
whole and ragged, so that the loop of four stages (eight steps where two groups of waves share them) runs never, once and
more often, with 0 to 3 stages after it. The library tells which tile a size takes. Bounds as in test_gpu_fp4_gemm.py."""

from __future__ import annotations

import pytest
import torch

from fp4_choice import choice
from fp4_helpers import activations, random_weight, weight
from test_gpu_fp4_gemm import _check, _run

pytestmark = pytest.mark.gpu

TILES = [  # rows in 8 bits, gate/up, M, N, tile
    (False, False, 40, 14330, (32, 128)), (False, False, 777, 1500, (64, 128)), (False, False, 300, 8190, (64, 256)),
    (False, True, 33, 6150, (32, 128)), (False, True, 70, 6150, (64, 128)), (False, True, 777, 1500, (64, 256)),
    (True, False, 40, 14330, (32, 128)), (True, False, 777, 1500, (64, 128)), (True, False, 777, 6150, (128, 256)),
    (True, True, 33, 6150, (32, 128)), (True, True, 70, 6150, (64, 128)), (True, True, 300, 8190, (128, 256))]
DEPTHS = [32, 160, 384, 416, 608, 768, 896, 992, 1056, 1280, 1408, 1536, 1824, 1920, 2048]


@pytest.mark.parametrize("k", DEPTHS)
@pytest.mark.parametrize("rows,glu,m,n,tile", TILES)
def test_products(pkg, rows, glu, m, n, tile, k):
    assert choice(pkg, m, n, k, rows, glu) == (*tile, 1)
    _check(pkg, m, n, k, rows, glu, seed=k)


@pytest.mark.parametrize("k", [896, 1408, 1920])
@pytest.mark.parametrize("rows,glu,m,n,tile", TILES)
def test_equal_calls_give_equal_bits(pkg, rows, glu, m, n, tile, k):
    """Over weights and rows of which each fresh call finds other ones' remains in LDS."""
    x, other = activations(m, k, 1).cuda(), activations(m, k, 2).cuda()
    w = weight(pkg, *random_weight(2 * n if glu else n, k, 3), glu)
    want = _run(pkg, x, w, rows, glu)
    for _ in range(20):
        _run(pkg, other, w, rows, glu)
        assert torch.equal(_run(pkg, x, w, rows, glu), want)


# The sizes of a 7-billion-parameter model's MLP cut in two, and K split into ranges whose last is cut short.
@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k,glu", [(300, 2048, 5504, False), (777, 2048, 5504, False), (100, 2048, 5504, False),
                                       (100, 1030, 15232, False), (300, 1030, 15232, False), (130, 530, 15232, True),
                                       (700, 1030, 15232, True), (300, 2050, 15136, False)])
def test_deep_products(pkg, m, n, k, glu, rows):
    _check(pkg, m, n, k, rows, glu, seed=m)
