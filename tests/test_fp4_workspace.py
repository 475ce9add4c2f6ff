"""What a 4-bit product needs as workspace, by the fields that its header names; no GPU."""

from __future__ import annotations

import pytest

from test_fp4_args import E_SHAPE, E_WORKSPACE, FAKE, ROWS8, _gemm, _gemm_args

SPLIT = dict(m=200, n=4096, y_stride=4096, k=14336, x_stride=14336)


def _bytes(pkg, **changes):
    return pkg.library().lse_fp4_gemm_workspace_bytes(_gemm_args(changes))


@pytest.mark.parametrize("glu", [0, 1])
@pytest.mark.parametrize("rows", [{}, dict(x_scales=FAKE)], ids=["bf16", "fp8"])
def test_only_the_sizes_and_the_kind_of_rows_count(pkg, glu, rows):
    """The same bytes whatever stands in the other fields, and enough for the call."""
    none = dict(x=None, x_stride=0, s_stride=0, codes=None, scales=None, y=None, y_stride=0)
    for m in (1, 60, 96, 200, 300, 1000):
        sizes = dict(m=m, n=4096, k=14336, glu=glu, **rows)
        need = _bytes(pkg, **sizes, **none)
        assert need == _bytes(pkg, **sizes) >= 0
        if need:
            call = {**SPLIT, **sizes, "s_stride": 448 if rows else 0}
            assert _gemm(pkg, call, FAKE, need - 1) == E_WORKSPACE


def test_rows_in_8_bits_have_a_plan_of_their_own(pkg):
    assert _bytes(pkg, m=200, n=4096, k=14336, glu=1) == 0
    assert _bytes(pkg, **{**ROWS8, **dict(m=200, n=4096, k=14336, glu=1)}) == 4 * 200 * 2 * 4096 * 4


@pytest.mark.parametrize("glu", [-1, 2, 1 << 32])
def test_the_products_kinds_are_refused_alike(pkg, glu):
    assert _bytes(pkg, glu=glu) == -1 and _bytes(pkg, m=0, glu=glu) == -1
    assert _gemm(pkg, dict(glu=glu)) == E_SHAPE


def test_tiles_sizes_are_of_weights_that_can_be_packed(pkg):
    lib = pkg.library()
    for size in (lib.lse_fp4_codes_bytes, lib.lse_fp4_scales_bytes):
        assert size(100, 544, 1) > 0 and size(0, 544, 1) == size(100, 0, 0) == 0
        assert size(100, 544, 2) == size(100, 544, -1) == size(99, 544, 1) == size((1 << 31) - 16, 544, 0) == -1
