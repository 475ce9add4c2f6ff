"""Rows whose positions no table holds: the append drops their k and v, and its q has what `rope` gives."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fp8_kv_helpers import bf16_rows, i32, plan_of, pool_to_dev, pool_to_host, random_pool, same_pool, to_dev
from helpers import bf16_bits
from oracle import kv_cache as kv

pytestmark = pytest.mark.gpu


def _append_into(pkg, pool, q, k, v, cos, sin, q_out, plan, most):
    """Through the C entry point into a caller's q_out; cos None: no rotation."""
    from llm_serving_engine_amd import _lib

    table, qo, qs, ql = plan
    tokens, h, d = q.shape
    n_kv, per = pool.k.shape[1:3]
    tables = (0, 0, 0) if cos is None else (cos.data_ptr(), sin.data_ptr(), len(cos))
    args = _lib.APPEND_KV_FP8_ARGS.pack(
        q.data_ptr(), h * d, d, k.data_ptr(), n_kv * d, d, v.data_ptr(), n_kv * d, d, *tables, q_out.data_ptr(),
        pool.k.data_ptr(), pool.v.data_ptr(), pool.k.stride(0), pool.scales.data_ptr(), pool.scales.stride(0),
        len(pool.k), 16 * per, table.data_ptr(), table.stride(0), table.shape[1], qo.data_ptr(), qs.data_ptr(),
        ql.data_ptr(), len(ql), tokens, most, h, n_kv, d, 0 if cos is None else 2 * cos.shape[1], 0)
    status = pkg.library().lse_append_kv_fp8(args, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status == 0


@pytest.mark.parametrize("turned", [True, False])
@pytest.mark.parametrize("news", [
    [(5, 3), (3, -2), (40, -17), (17, -33), (1, 9)], [(1, -1), (1, 30), (1, -16), (1, -2147483648)],
    [(20, -1000), (1, 5), (2, 2147483640), (33, -33)]])
def test_every_row_of_an_entry_is_rotated(pkg, dev, news, turned):
    """Entries of negative offsets, and of ones past any table, among ordinary ones: every q row is `rope`'s at its
    position (NaN where the tables have none), k and v of the ordinary ones alone are written."""
    rng = np.random.default_rng(len(news))
    h, h_kv, d = 4, 2, 64
    case = plan_of(rng, [(n, min(max(o, 0), 60), n) for n, o in news], 16)
    case["qo"] = np.array([o for _, o in news], np.int32)
    tokens = int(case["ql"].sum())
    q, k, v = (bf16_rows(rng, tokens, heads, d) for heads in (h, h_kv, h_kv))
    cos, sin = pkg.ops.rope_table(80, d, device=dev)
    pos = np.concatenate([np.arange(o, o + n) for n, o in news])
    pos = np.where((pos < 0) | (pos >= 80), -1, pos)
    host = random_pool(rng, case["blocks"], 16, h_kv, d)
    pool = pool_to_dev(pkg, host, dev)
    q_out = torch.full((tokens, h, d), 7.0, dtype=torch.bfloat16, device=dev)
    plan = [i32(case[n], dev) for n in ("table", "qo", "qs", "ql")]
    qd, kd, vd = (to_dev(x, dev) for x in (q, k, v))
    tables = (cos, sin) if turned else (None, None)
    _append_into(pkg, pool, qd, kd, vd, *tables, q_out, plan, max(n for n, _ in news))
    want = pkg.ops.rope(qd, None, cos, sin, i32(pos, dev))[0] if turned else qd
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(q_out), nan)
    np.testing.assert_array_equal(bf16_bits(q_out[~nan]), bf16_bits(want[~nan]))
    assert not turned or nan.any()
    if turned:
        k = kv.rotate(k, cos.cpu().numpy(), sin.cpu().numpy(), np.maximum(pos, 0), False)
    kv.append(host, k, v, case["table"], case["qo"], case["qs"], case["ql"], 16)
    same_pool(pool_to_host(pool), host)
