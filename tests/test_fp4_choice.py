"""Which kernel a product with a 4-bit weight runs, as the library itself tells: literal sizes on both sides of bounds;
no GPU."""

from __future__ import annotations

import ctypes

import pytest

from fp4_choice import choice
from test_fp4_args import E_ALIGN, E_NULL, E_RANGE, E_SHAPE, _gemm_args

# (token rows from which on, up to which, tile rows, tile columns, ranges of K) for a weight and a kind of rows.
BF16, FP8 = False, True


@pytest.mark.parametrize("n,k,rows,glu,spans", [
    (4096, 4096, BF16, 0, [(1, 4, 0, 16, 1), (5, 7, 0, 32, 1), (17, 32, 0, 32, 1), (33, 128, 0, 64, 1),
                           (129, 256, 32, 128, 1), (257, 512, 64, 128, 1), (513, 1024, 64, 256, 1)]),
    (4096, 14336, BF16, 0, [(17, 32, 0, 32, 1), (33, 64, 32, 128, 4), (65, 128, 64, 128, 4), (129, 170, 64, 256, 4),
                            (171, 227, 64, 128, 2), (302, 512, 64, 128, 1), (729, 1024, 64, 256, 1)]),
    (14336, 4096, BF16, 1, [(1, 4, 0, 32, 1), (5, 16, 0, 64, 1), (17, 32, 32, 128, 1), (33, 64, 64, 128, 1),
                            (65, 128, 64, 256, 1), (321, 4096, 64, 256, 1)]),
    (4096, 4096, FP8, 0, [(1, 8, 0, 16, 1), (9, 15, 0, 32, 1), (33, 64, 0, 64, 1), (129, 256, 32, 128, 1),
                          (257, 1024, 64, 128, 1), (1025, 2048, 128, 256, 1)]),
    (4096, 14336, FP8, 0, [(33, 64, 0, 64, 1), (65, 170, 64, 128, 4), (171, 256, 64, 128, 2), (257, 446, 128, 256, 4),
                           (447, 512, 64, 128, 1), (513, 1024, 128, 256, 2), (1025, 2048, 128, 256, 1)]),
    (14336, 4096, FP8, 1, [(1, 8, 0, 32, 1), (9, 32, 32, 128, 1), (33, 128, 64, 128, 1), (129, 4096, 128, 256, 1)])])
def test_which_kernel(pkg, n, k, rows, glu, spans):
    for first, last, *want in spans:
        assert choice(pkg, first, n, k, rows, glu) == choice(pkg, last, n, k, rows, glu) == tuple(want), (first, last)


def test_every_kernel_is_reached(pkg):
    for rows in (BF16, FP8):
        for glu in (0, 1):
            got = {choice(pkg, m, n, k, rows, glu)[:2] for m in (1, 5, 13, 33, 70, 150, 300, 777, 2048)
                   for n in (100, 1500, 4096, 6150, 14336) for k in (544, 4096, 14336)}
            tiles = {(32, 128), (64, 128), (128, 256) if rows else (64, 256)}
            assert got == tiles | {(0, 16 * w) for w in ((2, 4) if glu else (1, 2, 4))}


def test_workspaces_are_the_ranges_sums(pkg):
    for m, n, k, rows, glu in [(200, 4096, 14336, BF16, 0), (40, 4096, 14336, BF16, 0), (130, 530, 28704, FP8, 1),
                               (2048, 4096, 4096, FP8, 0), (300, 1030, 14336, BF16, 1)]:
        splits = choice(pkg, m, n, k, rows, glu)[2]
        nbytes = pkg.library().lse_fp4_gemm_workspace_bytes(_gemm_args(dict(m=m, n=n, k=k, glu=glu, x_scales=16 if rows else None)))
        assert nbytes == (splits * m * 16 * (1 + glu) * -(-n // 16) * 4 if splits > 1 else 0)


def test_refusals(pkg):
    fn = pkg.library().lse_fp4_gemm_choice
    v = [ctypes.c_int64(-1) for _ in range(3)]
    out = [ctypes.byref(x) for x in v]
    assert fn(None, *out) == fn(_gemm_args({}), out[0], None, out[2]) == E_NULL
    assert fn(_gemm_args(dict(glu=2)), *out) == fn(_gemm_args(dict(m=-1)), *out) == E_SHAPE
    assert fn(_gemm_args(dict(k=40)), *out) == E_ALIGN and fn(_gemm_args(dict(k=1 << 22)), *out) == E_RANGE
    assert [x.value for x in v] == [-1] * 3
    for empty in (dict(m=0), dict(n=0), dict(k=0)):
        assert fn(_gemm_args(empty), *out) == 0 and [x.value for x in v] == [0] * 3
