"""Which kernel a 4-bit product takes, as the library tells it."""

from __future__ import annotations

import ctypes


def choice(pkg, m: int, n: int, k: int, rows: bool, glu: bool) -> tuple[int, int, int]:
    """(token rows of a tile or 0, weight rows of a tile, ranges of K); rows: in 8 bits."""
    from llm_serving_engine_amd import _lib

    args = _lib.FP4_GEMM_ARGS.pack(0, 0, 16 if rows else 0, 0, 0, 0, 0, 0, m, n, k, int(glu))
    out = [ctypes.c_int64(-1) for _ in range(3)]
    assert pkg.library().lse_fp4_gemm_choice(args, *map(ctypes.byref, out)) == 0
    return tuple(v.value for v in out)
