"""Products with 4-bit weights on the GPU against the definition in 64 bits.

Tolerances. S = sum_k |x w| of an output, y the output in 64 bits. Rounding to bf16: 2^-8 |y|. fp32 sums of K exact
products in any order: at most K 2^-24 S. With rows in 8 bits the matrix instruction cuts the products of eight
consecutive k off 13 bits below the largest of them, which itself is whole: seven lose less than 2^-13 of the eight's
sum of magnitudes, 7 2^-13 S < 2^-10 S. Gate/up: h = silu(g) u, with |silu(g)| <= |g|, |silu'| <= 1.1 and the same
bounds on g and u; the exponential and the quotient add 2^-20 |h|.
"""

from __future__ import annotations

import pytest
import torch

from fp4_helpers import E8, F8, activations, few_ones, random_weight, rows8, weight
from oracle import fp4 as ora

pytestmark = pytest.mark.gpu


def _bound(y, s, k, rows):
    return 2.0 ** -8 * y.abs() + s * (k * 2.0 ** -24 + (2.0 ** -10 if rows else 0.0))


def _glu_bound(g, sg, u, su, k, rows):
    dg, du = sg * (k * 2.0 ** -24 + (2.0 ** -10 if rows else 0)), su * (k * 2.0 ** -24 + (2.0 ** -10 if rows else 0))
    h = ora.glu(g, u)
    return (2.0 ** -8 + 2.0 ** -20) * h.abs() + 1.1 * dg * (u.abs() + du) + g.abs() * du


def _run(pkg, x, w, rows, glu):
    ops = pkg.ops
    if rows:
        return (ops.w4a8_glu if glu else ops.w4a8_linear)(ops.quantize_rows_fp8(x.cuda()), w)
    return (ops.w4a16_glu if glu else ops.w4a16_linear)(x.cuda(), w)


def _values(x, rows):
    return ora.row_values(*ora.quantize_rows(x)) if rows else x.double()


def _check(pkg, m, n, k, rows, glu, seed=0):
    code, byte = random_weight(2 * n if glu else n, k, seed)
    x = activations(m, k, seed + 1)
    y = _run(pkg, x, weight(pkg, code, byte, glu), rows, glu)
    assert y.shape == (m, n) and y.dtype == torch.bfloat16
    values, w = _values(x, rows).cuda(), ora.weight_values(code, byte).cuda()
    if glu:
        (g, sg), (u, su) = (ora.product(values, part) for part in (w[:n], w[n:]))
        want, bound = ora.glu(g, u), _glu_bound(g, sg, u, su, k, rows)
    else:
        want, s = ora.product(values, w)
        bound = _bound(want, s, k, rows)
    off = (y.double() - want).abs()
    assert bool((off <= bound).all()), f"{int((off > bound).sum())} of {off.numel()} off, worst {float((off / bound).max())}"


SIZES = [(1, 16, 32), (1, 1, 512), (2, 40, 4096), (3, 17, 96), (4, 256, 1024), (5, 33, 160), (7, 1000, 544),
         (8, 64, 14336), (9, 130, 2048), (15, 257, 1056), (16, 512, 512), (17, 96, 640), (31, 48, 4128), (33, 300, 288),
         (64, 128, 2080), (65, 64, 1024), (100, 1030, 608), (129, 272, 4096), (300, 520, 1312), (513, 768, 256)]


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(pkg, m, n, k, rows):
    _check(pkg, m, n, k, rows, False)


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_glu(pkg, m, n, k, rows):
    _check(pkg, m, n, k, rows, True)


# The widest tiles, at their edges in every direction.
LARGE = [(1000, 6150, 1184), (2100, 3601, 160), (700, 3601, 2080), (1023, 2070, 96), (301, 6150, 672)]


@pytest.mark.parametrize("glu", [False, True], ids=["linear", "glu"])
@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", LARGE)
def test_large(pkg, m, n, k, rows, glu):
    _check(pkg, m, n, k, rows, glu)


@pytest.mark.parametrize("m,n,k", [(1, 300, 4128), (13, 100, 1184), (70, 333, 2048), (300, 500, 1600), (1000, 6150, 1184)])
@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
def test_every_place_exactly(pkg, m, n, k, rows):
    """Five values of a row, so every output is a multiple of 1/8 below 32: exact in bf16, whatever the order."""
    g = torch.Generator().manual_seed(m)
    code, byte = torch.randint(0, 16, (n, k), generator=g), torch.randint(126, 128, (n, k // 32), generator=g)
    x = few_ones(m, k, 5, m + 1)
    w = weight(pkg, code, byte)
    want = x.double() @ ora.weight_values(code, byte).t()
    if rows:
        xb = torch.randint(126, 128, (m, k // 32), generator=g)
        held = pkg.ops.Fp8Rows(x.to(F8).cuda(), xb.to(torch.uint8).view(E8).cuda())
        want = ora.row_values(x.double(), xb) @ ora.weight_values(code, byte).t()
        y = pkg.ops.w4a8_linear(held, w)
    else:
        y = pkg.ops.w4a16_linear(x.to(torch.bfloat16).cuda(), w)
    assert torch.equal(y.double().cpu(), want)
