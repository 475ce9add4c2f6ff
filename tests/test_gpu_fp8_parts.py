"""The row-tiled kernel over the 8-bit cache where its items are cut into parts, and in the calls around it: layouts,
rows of nobody, padded buckets, streams, scales, infinite scores. Tolerance as in test_gpu_fp8_attention.py; what a
call runs is asserted by the library's own choice."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fp8_attention_helpers import attend_into, choice_of
from fp8_kv_helpers import (attend, attend_args, attention_case, attention_golden, check_attention, pool_to_dev)
from helpers import bf16_bits, to_bf16_tensor
from oracle import kv_cache as kv
from oracle import numerics as ora

pytestmark = pytest.mark.gpu


def _decodes(n, ctx):
    return [(1, ctx - 1 - 13 * i, ctx - 13 * i) for i in range(n)]


# (entries, heads, K/V heads, parts): chunks beside 40 decode rows in two and three parts, and alone in two to sixteen;
# where contexts differ, the short ones' items have fewer.
CUT = [
    ([(400, 900, 1300)] + _decodes(40, 610), 32, 8, 2),
    ([(440, 1000, 1440), (30, 200, 230)] + _decodes(40, 620), 32, 8, 2),
    ([(300, 1700, 2000)] + _decodes(40, 700), 24, 8, 3),
    ([(600, 1900, 2500)], 32, 8, 3),
    ([(420, 6080, 6500)], 16, 4, 9),
    ([(380, 6080, 6460), (40, 700, 740), (50, 0, 50), (1, 3000, 3001)], 16, 4, 8),
    ([(330, 8000, 8330), (130, 2000, 2130)], 8, 2, 16),
]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("entries,h,h_kv,parts", CUT)
def test_items_in_parts(pkg, dev, entries, h, h_kv, parts, d):
    case = attention_case(len(entries) * parts + d, entries, h=h, h_kv=h_kv, d=d, block_size=32)
    assert choice_of(pkg, case)[:2] == (True, parts)
    check_attention(pkg, dev, case, f"{parts} parts")


def test_parts_end_with_the_context(pkg, dev):
    """Contexts shorter than the rows' positions: later items of fewer tiles than parts, one of none."""
    case = attention_case(5, [(400, 900, 1300)] + _decodes(40, 610), block_size=32)
    for ctx in (1299, 385, 383, 64, 0):
        case["ctx"][0] = ctx
        assert choice_of(pkg, case)[1] == 2
        o = check_attention(pkg, dev, case, f"context {ctx}")
        assert ctx > 0 or not o[:, :400].any()


LAYOUTS = [([(400, 900, 1300)] + _decodes(40, 610), 32, 8, 128, 2),  # in parts
           ([(150, 450, 600), (64, 0, 64), (1, 500, 501)], 136, 34, 64, 1),  # whole
           ([(300, 17000, 17300), (1, 3000, 3001), (2, 7, 9)], 4, 1, 64, 16)]  # in parts beside split decode rows


@pytest.fixture(params=LAYOUTS, ids=["parts", "whole", "split"])
def layout(request, pkg, dev):
    entries, h, h_kv, d, parts = request.param
    case = attention_case(h + parts, entries, h=h, h_kv=h_kv, d=d, block_size=32)
    assert choice_of(pkg, case)[:2] == (True, parts)
    return case, attend(pkg, dev, case)


def test_token_major_rows_and_two_streams(pkg, dev, layout):
    """q as a slice of a stacked projection; two calls in flight at once."""
    case, want = layout
    h, tokens, d = case["q"].shape
    stacked = torch.zeros(tokens, h + 4, d, dtype=torch.bfloat16, device=dev)
    stacked[:, :h] = to_bf16_tensor(case["q"], dev).transpose(0, 1)
    pool, plan = pool_to_dev(pkg, case["pool"], dev), attend_args(case, dev)
    q = stacked[:, :h].transpose(0, 1)
    torch.cuda.synchronize()
    got = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(pkg.ops.paged_attention_fp8(q, pool, *plan, int(case["ql"].max())))
    torch.cuda.synchronize()
    for o in got:
        assert o.stride(1) == h * d
        np.testing.assert_array_equal(bf16_bits(o), want)


def test_rows_of_no_entry_are_left_alone(pkg, dev, layout):
    """Rows before, between and behind the entries' keep what the caller's o held, whose heads lie far apart."""
    case, want = layout
    h, tokens, d = case["q"].shape
    gap = 5
    at = np.concatenate([np.arange(s, s + n) + gap * (e + 1) for e, (s, n) in enumerate(zip(case["qs"], case["ql"]))])
    total = tokens + gap * (len(case["ql"]) + 1)
    q = torch.zeros(h, total, d, dtype=torch.bfloat16, device=dev)
    q[:, at] = to_bf16_tensor(case["q"], dev)
    assert choice_of(pkg, dict(case, q=np.zeros((h, total, d), np.uint16))) == choice_of(pkg, case)
    table, ctx, qo, qs, ql = attend_args(case, dev)
    starts = qs + gap * torch.arange(1, len(qs) + 1, device=dev, dtype=torch.int32)
    wide = torch.full((total, h, 2 * d), 7.0, dtype=torch.bfloat16, device=dev)
    o = wide[..., :d].transpose(0, 1)
    attend_into(pkg, q, pool_to_dev(pkg, case["pool"], dev), (table, ctx, qo, starts, ql), int(case["ql"].max()), o)
    np.testing.assert_array_equal(bf16_bits(o[:, at]), want)
    assert (o[:, np.setdiff1d(np.arange(total), at)] == 7.0).all() and (wide[..., d:] == 7.0).all()


def test_rows_outside_the_calls_are_left_alone(pkg, dev, layout):
    """The first entry starts three rows before the call's, the last one behind them: a buffer's rows around the call's
    keep what they held, the others are those of the same tokens inside."""
    case, _ = layout
    h, tokens, d = case["q"].shape
    n0, last = int(case["ql"][0]), int(case["qs"][-1])
    moved = case["q"].copy()
    moved[:, 3:n0] = case["q"][:, :n0 - 3]  # token m of the first entry reads row m - 3
    want = attend(pkg, dev, dict(case, q=moved))
    lead = 8
    buffer = torch.full((h, lead + tokens + 8, d), 7.0, dtype=torch.bfloat16, device=dev)
    q, o = torch.zeros_like(buffer), buffer[:, lead:lead + tokens]
    q[:, lead:lead + tokens] = to_bf16_tensor(case["q"], dev)
    table, ctx, qo, qs, ql = attend_args(case, dev)
    qs[0], qs[-1] = -3, tokens
    attend_into(pkg, q[:, lead:lead + tokens], pool_to_dev(pkg, case["pool"], dev), (table, ctx, qo, qs, ql),
                int(case["ql"].max()), o)
    np.testing.assert_array_equal(bf16_bits(o[:, :n0 - 3]), want[:, 3:n0])
    np.testing.assert_array_equal(bf16_bits(o[:, n0:last]), want[:, n0:last])
    assert (o[:, n0 - 3:n0] == 7.0).all() and (o[:, last:] == 7.0).all()
    assert (buffer[:, :lead] == 7.0).all() and (buffer[:, lead + tokens:] == 7.0).all()


def test_padded_buckets(pkg, dev, layout):
    """Entries of no tokens, a larger max_q_len and rows behind the last, under the same table width: the bits of the
    call without them where the choice comes out alike, else within the tolerance."""
    case, want = layout
    tokens = case["q"].shape[1]
    for more, most in ((0, int(case["ql"].max()) + 70), (3, None), (30, None)):
        pad = dict(case, **{n: np.concatenate([case[n], np.zeros(more, np.int32)]) for n in ("ctx", "qo", "qs", "ql")})
        pad["table"] = np.concatenate([case["table"], np.full((more, case["table"].shape[1]), -1, np.int32)])
        pad["q"] = np.concatenate([case["q"], np.full_like(case["q"][:, :7], 0x7fc0)], 1)
        if choice_of(pkg, pad, most) == choice_of(pkg, case) and choice_of(pkg, case)[2] == 0:
            np.testing.assert_array_equal(attend(pkg, dev, pad, most)[:, :tokens], want)
        else:
            o = attend(pkg, dev, pad, most)[:, :tokens]
            golden, covered, vmax = attention_golden(case)
            ok, msg = ora.attention_within_tolerance(o, golden, vmax, covered)
            assert ok, msg


# The key-streaming kernel alone, its split form, and the three above.
SCALED = [([(1, 699, 700), (40, 300, 340), (5, 0, 5)], 8, 2, 128, 0),
          ([(1, 5999, 6000), (3, 40, 43)], 8, 2, 64, 0), *LAYOUTS]


@pytest.mark.parametrize("entries,h,h_kv,d,parts", SCALED)
def test_zero_and_negative_scales(pkg, dev, entries, h, h_kv, d, parts):
    """A negative scale is that of -q: the same products, exactly. Zero is the mean of what a row sees, the bits of
    q = 0. Against fp64 as well."""
    case = attention_case(h * d + parts, entries, h=h, h_kv=h_kv, d=d, block_size=32)
    assert choice_of(pkg, case)[:2] == (parts > 0, parts)
    q, pool, plan = to_bf16_tensor(case["q"], dev), pool_to_dev(pkg, case["pool"], dev), attend_args(case, dev)
    most = int(case["ql"].max())
    o, ref = torch.empty_like(q), torch.empty_like(q)
    k, v = (ora.f32_to_bf16_bits(x.astype(np.float32)) for x in kv.unpack(case["pool"], case["bs"]))
    vmax = float(np.abs(ora.bf16_bits_to_f32(v)).max())
    for scale, like, like_scale in ((-0.07, -q, 0.07), (0.0, torch.zeros_like(q), 0.07), (0.01, q, 0.01)):
        attend_into(pkg, q, pool, plan, most, o, scale)
        attend_into(pkg, like, pool, plan, most, ref, like_scale)
        np.testing.assert_array_equal(bf16_bits(o), bf16_bits(ref))
        golden, covered = ora.paged_attention_golden(case["q"], k, v, case["table"], case["ctx"], case["qo"],
                                                     case["qs"], case["ql"], case["bs"], scale)
        ok, msg = ora.attention_within_tolerance(bf16_bits(o), golden, vmax, covered)
        assert ok, f"scale {scale}: {msg}"


@pytest.mark.parametrize("entries,h,h_kv,d,parts", SCALED)
def test_infinite_scores(pkg, dev, entries, h, h_kv, d, parts):
    """A key of score -inf is left out, one of +inf makes the rows that see it NaN, and no other row: dim 0 of the
    keys is zero but for key 3 of entry 0, and that of one row of q is so large that the product leaves fp32."""
    case = attention_case(h * d + 7, entries, h=h, h_kv=h_kv, d=d, block_size=32)
    assert choice_of(pkg, case)[:2] == (parts > 0, parts)
    k, v, s = (a.copy() for a in case["pool"])
    for slot in range(16):
        k[..., kv.k_index(slot, 0, d)] = 0
    block = case["table"][0, 0]
    k[block, :, 0, kv.k_index(3, 0, d)] = 0x7e  # 448 scales
    s[block, :, 0, 0] = 127
    case["pool"] = (k, v, s)
    rows = [int(case["ql"][0]) - 1, int(case["ql"][0]) // 2]  # of entry 0, both beyond key 3
    q = ora.bf16_bits_to_f32(case["q"]).copy()
    q[..., 0] = 0.0
    case["q"] = ora.f32_to_bf16_bits(q)
    want = attend(pkg, dev, case)
    big = float(torch.finfo(torch.bfloat16).max)
    q[:, rows, 0] = -big
    case["q"] = ora.f32_to_bf16_bits(q)
    golden, covered, vmax = attention_golden(case)  # in fp64 its probability is 0
    o = attend(pkg, dev, case)
    ok, msg = ora.attention_within_tolerance(o, golden, vmax, covered)
    assert ok, msg
    others = np.setdiff1d(np.arange(q.shape[1]), rows)
    np.testing.assert_array_equal(o[:, others], want[:, others])
    q[:, rows, 0] = big
    case["q"] = ora.f32_to_bf16_bits(q)
    o = attend(pkg, dev, case)
    assert np.isnan(ora.bf16_bits_to_f32(o[:, rows])).all()
    ok, msg = ora.attention_within_tolerance(o[:, others], golden[:, others], vmax, covered[others])
    assert ok, msg


def test_a_row_of_infinities_only(pkg, dev):
    """Every key that a row sees left out: zeros, in either kernel, as without a context."""
    for entries, h, h_kv, d, parts in SCALED:
        case = attention_case(h + d, entries, h=h, h_kv=h_kv, d=d, block_size=32)
        k, v, s = (a.copy() for a in case["pool"])
        for slot in range(16):
            k[..., kv.k_index(slot, 0, d)] = 0x7e
        s[..., 0] = 127
        case["pool"] = (k, v, s)
        q = ora.bf16_bits_to_f32(case["q"]).copy()
        row = int(case["ql"][0]) - 1
        q[:, row, 0] = -float(torch.finfo(torch.bfloat16).max)
        case["q"] = ora.f32_to_bf16_bits(q)
        o = attend(pkg, dev, case)
        assert not ora.bf16_bits_to_f32(o[:, row]).any()
        assert np.isfinite(ora.bf16_bits_to_f32(o)).all()
        assert choice_of(pkg, case)[:2] == (parts > 0, parts)


def test_items_in_parts_replay_from_a_graph(pkg, dev):
    """Two parts, captured twice over workspaces of the graphs' pool, replayed in turn with eager calls between."""
    case = attention_case(9, LAYOUTS[0][0], block_size=32)
    pool, q, plan = pool_to_dev(pkg, case["pool"], dev), to_bf16_tensor(case["q"], dev), attend_args(case, dev)
    call = lambda: pkg.ops.paged_attention_fp8(q, pool, *plan, 400)  # noqa: E731
    call()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call()))
    for _ in range(3):
        for graph, o in graphs:
            q.mul_(-1.25)
            graph.replay()
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(o, want)


def test_another_plan_of_the_same_sizes(pkg, dev):
    """A captured call of two parts over other contexts, offsets and lengths than it was captured with."""
    case = attention_case(11, LAYOUTS[0][0], block_size=32)
    pool, q = pool_to_dev(pkg, case["pool"], dev), to_bf16_tensor(case["q"], dev)
    table, ctx, qo, qs, ql = attend_args(case, dev)
    call = lambda: pkg.ops.paged_attention_fp8(q, pool, table, ctx, qo, qs, ql, 400)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call()
    for n, before in ((100, 300), (31, 1200), (0, 0), (399, 0)):
        ql[0], qo[0], ctx[0] = n, before, n + before
        now = dict(case, ql=ql.cpu().numpy(), qo=qo.cpu().numpy(), ctx=ctx.cpu().numpy())
        graph.replay()
        torch.cuda.synchronize()
        golden, covered, vmax = attention_golden(now)
        ok, msg = ora.attention_within_tolerance(bf16_bits(o), golden, vmax, covered)
        assert ok, f"{n} behind {before}: {msg}"
