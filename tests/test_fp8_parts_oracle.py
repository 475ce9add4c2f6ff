"""That the tolerance of the row-tiled kernel's tests tells a part left out: the fp64 result without one part's keys is
outside it. No GPU."""

from __future__ import annotations

import numpy as np
import pytest

from fp8_kv_helpers import attention_case
from oracle import kv_cache as kv
from oracle import numerics as ora


@pytest.mark.parametrize("n,before,parts", [(400, 900, 2), (300, 1700, 3), (420, 6080, 9), (300, 8000, 16)])
def test_a_part_left_out_is_told(n, before, parts):
    g, ctx = 4, n + before
    case = attention_case(n + parts, [(n, before, ctx)], h=g, h_kv=1, block_size=32)
    k, v = (x.reshape(-1, 32, 128) for x in kv.unpack(case["pool"], 32))
    k, v = (x[case["table"][0]].reshape(-1, 128)[:ctx] for x in (k, v))
    rows = n - 128 // g + np.arange(128 // g)  # the last item's
    q = ora.bf16_bits_to_f32(case["q"])[:, rows].astype(np.float64)
    at = np.arange(ctx)
    score = np.einsum("hmd,nd->hmn", q, k) / np.sqrt(128)
    score = np.where(at[None] <= (before + rows)[:, None], score, -np.inf)

    def result(keep):
        s = np.where(keep, score, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        return p @ v / p.sum(-1, keepdims=True)

    golden, vmax = result(at >= 0), float(np.abs(v).max())
    assert ora.attention_within_tolerance(ora.f32_to_bf16_bits(golden.astype(np.float32)), golden, vmax)[0]
    tiles = -(-ctx // 64)
    for part in range(parts):
        lo, hi = (64 * (tiles * p // parts) for p in (part, part + 1))
        bad = result((at < lo) | (at >= hi))
        assert not ora.attention_within_tolerance(ora.f32_to_bf16_bits(bad.astype(np.float32)), golden, vmax)[0], part
