"""Paged attention over the 8-bit K/V cache on the GPU against the fp64 oracle on the values the cache stands
for. Tolerance (`fp8_kv_helpers.check_attention`): bf16 probabilities and a bf16 output, as for the bf16 cache."""

from __future__ import annotations

import re
from pathlib import Path

import numpy as np
import pytest
import torch

from fp8_kv_helpers import (attend, attend_args, attention_case, attention_golden, bf16_rows, check_attention,
                            i32, pool_to_dev, to_dev)
from helpers import bf16_bits, to_bf16_tensor
from oracle import kv_cache as kv
from oracle import numerics as ora

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctxs", [[1, 2, 15, 16, 17], [63, 64, 65, 255, 256, 257], [1023, 1024, 1025, 3, 700],
                                  [1279, 1281, 2047, 2050, 4095]])
def test_decode_rows(pkg, dev, d, ctxs):
    """One row a sequence at every edge of a group, a tile, a window and a round of four chunks."""
    check_attention(pkg, dev, attention_case(d + len(ctxs), [(1, c - 1, c) for c in ctxs], d=d), f"{ctxs}")


@pytest.mark.parametrize("h,h_kv", [(8, 8), (16, 8), (24, 8), (40, 8), (32, 2), (16, 1), (10, 2), (7, 1), (26, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_head_groupings(pkg, dev, h, h_kv, d):
    """1 to 16 query heads per K/V head, those that do not divide a tile's 16 rows among them."""
    entries = [(5, 10, 15), (1, 40, 41), (20, 0, 20), (7, 600, 607), (1, 1300, 1301)]
    check_attention(pkg, dev, attention_case(h * d + h_kv, entries, h=h, h_kv=h_kv, d=d), f"{h} over {h_kv}")


@pytest.mark.parametrize("block_size", [16, 32, 48, 64, 80, 256])
def test_block_sizes(pkg, dev, block_size):
    entries = [(1, 500, 501), (9, 70, 79), (30, 0, 30), (1, 0, 1), (1, 47, 48), (2, 255, 257)]
    check_attention(pkg, dev, attention_case(block_size, entries, h=8, h_kv=2, block_size=block_size))


def test_mixed_chunks_and_decode(pkg, dev):
    entries = [(50, 0, 50), (33, 64, 97), (1, 200, 201), (7, 5, 12), (1, 0, 1), (129, 3, 132), (0, 9, 9),
               (1, 1500, 1501), (64, 1000, 1064)]
    check_attention(pkg, dev, attention_case(3, entries, h=24, h_kv=8, block_size=32), "mixed")


@pytest.mark.parametrize("d", [64, 128])
def test_prompts(pkg, dev, d):
    """Fresh prompts and later chunks of several hundred tokens."""
    entries = [(300, 0, 300), (257, 130, 387), (128, 1000, 1128), (1, 60, 61)]
    check_attention(pkg, dev, attention_case(20 + d, entries, h=8, h_kv=2, d=d), "prompts")


def test_contexts_end_before_the_rows_do(pkg, dev):
    """context_len below query_offset + q_len: later rows see no more than the context; none at all gives
    zeros; a context longer than the table is cut to it."""
    case = attention_case(30, [(20, 0, 20), (6, 40, 46), (1, 99, 100), (3, 10, 13)], h=8, h_kv=2)
    case["ctx"][:] = [7, 0, 50, 13]
    o = check_attention(pkg, dev, case)
    assert not o[:, 20:26].any()
    long = dict(case, ctx=case["ctx"].copy())
    case["ctx"][2], long["ctx"][2] = 100, 5000
    case["table"], long["table"] = (np.ascontiguousarray(c["table"][:, :7]) for c in (case, long))
    case["qo"][2] = long["qo"][2] = 111
    case["ctx"][2] = 112
    np.testing.assert_array_equal(attend(pkg, dev, long), attend(pkg, dev, case))


def test_nothing_outside_the_context_is_read_into_a_row(pkg, dev):
    """NaN codes in every slot behind a context and in every other block, NaN scales in groups behind it."""
    entries = [(1, 20, 21), (1, 63, 64), (40, 7, 47), (1, 300, 301), (18, 0, 18)]
    case = attention_case(31, entries, h=8, h_kv=2, block_size=32)
    want = attend(pkg, dev, case)
    k, v, s = (a.copy() for a in case["pool"])
    used = np.zeros((case["blocks"], 2, 16), bool)
    for e, (_, _, ctx) in enumerate(entries):
        for n in range(ctx):
            used[case["table"][e, n // 32], n % 32 // 16, n % 16] = True
    for b, sub, slot in np.argwhere(~used):
        dims = np.arange(128)
        k[b, :, sub, kv.k_index(slot, dims, 128)] = 127
        v[b, :, sub, kv.v_index(slot, dims, 128)] = 255
        if not used[b, sub].any():
            s[b, :, sub] = kv.NAN_SCALE
    np.testing.assert_array_equal(attend(pkg, dev, dict(case, pool=(k, v, s))), want)


def test_bad_blocks_reach_their_own_entry_only(pkg, dev):
    """A block outside the pool, and a NaN scale: the rows that see them are NaN, everything else as before."""
    case = attention_case(32, [(1, 99, 100), (1, 99, 100), (1, 1999, 2000), (4, 30, 34)], h=8, h_kv=2)
    want = attend(pkg, dev, case)
    bad = dict(case, table=case["table"].copy())
    bad["table"][0, 2], bad["table"][2, 100] = case["blocks"], -7
    pool = tuple(a.copy() for a in case["pool"])
    pool[2][case["table"][3, 0], :, 0, 0] = kv.NAN_SCALE
    o = ora.bf16_bits_to_f32(attend(pkg, dev, dict(bad, pool=pool)))
    assert np.isnan(o[:, [0, 2]]).all() and np.isnan(o[:, 3:7]).all()
    np.testing.assert_array_equal(ora.f32_to_bf16_bits(o[:, 1]), want[:, 1])


@pytest.mark.parametrize("q_scale", [0.0, 4.0, 2.0 ** 12, 2.0 ** 40, 2.0 ** -40])
def test_flat_and_peaked_scores(pkg, dev, q_scale):
    case = attention_case(33, [(1, 699, 700), (40, 300, 340)], h=8, h_kv=2, q_scale=q_scale)
    check_attention(pkg, dev, case, f"q x {q_scale}")


def _workspace(pkg, entries, tokens, h, h_kv, d, most, width, block_size):
    from llm_serving_engine_amd import _lib

    args = [0] * 26
    args[9], args[12], args[20:26] = block_size, width, (entries, tokens, most, h, h_kv, d)
    return pkg.library().lse_paged_attention_fp8_workspace_bytes(_lib.PAGED_ATTENTION_FP8_ARGS.pack(*args, 1.0))


def test_what_a_rows_bits_depend_on(pkg, dev):
    """A batch whose keys are split (few entries) and one whose are not: the same bits in a padded bucket
    under a table as wide as the pool, with a larger max_q_len, in another order; unsplit also among other
    entries."""
    rng = np.random.default_rng(34)
    ctxs = [2100, 1, 513, 300, 1030] + [int(c) for c in rng.integers(1, 400, 70)]
    case = attention_case(34, [(1, c - 1, c) for c in ctxs])
    width = case["table"].shape[1]
    size = lambda e: _workspace(pkg, e, e, 32, 8, 128, 1, width, 16)  # noqa: E731
    assert size(5) > 0 and size(75) == 0
    fields = ("table", "ctx", "qo", "qs", "ql")
    few = dict(case, q=case["q"][:, :5], **{n: case[n][:5] for n in fields})
    for c, entries, bucket in ((few, 5, 16), (case, 75, 96)):
        want = check_attention(pkg, dev, c, f"{entries} entries")
        wide = np.full((bucket, case["blocks"]), case["blocks"] - 1, np.int32)
        wide[:entries, :width] = c["table"]
        pad = dict(c, table=wide, **{n: np.concatenate([c[n], np.zeros(bucket - entries, np.int32)])
                                     for n in fields[1:]})
        np.testing.assert_array_equal(attend(pkg, dev, pad), want)
        np.testing.assert_array_equal(attend(pkg, dev, pad, most=9), want)
        back = dict(c, q=c["q"][:, ::-1].copy(), **{n: c[n][::-1].copy() for n in ("table", "ctx", "qo", "ql")})
        np.testing.assert_array_equal(attend(pkg, dev, back), want[:, ::-1])
    some = dict(case, q=case["q"][:, :68], **{n: case[n][:68] for n in fields})
    np.testing.assert_array_equal(attend(pkg, dev, some), want[:, :68])


@pytest.mark.parametrize("ctx", [2049, 32768, 32769, 70000])
def test_long_contexts(pkg, dev, ctx):
    """Split and unsplit, beside a short entry."""
    case = attention_case(ctx, [(1, ctx - 1, ctx), (2, 98, 100)], h=3, h_kv=1, d=64, block_size=64)
    assert _workspace(pkg, 2, 3, 3, 1, 64, 2, case["table"].shape[1], 64) > 0
    check_attention(pkg, dev, case, f"ctx {ctx} split")
    n = 520  # entries that fill the card, all but two of them empty
    pad = dict(case, **{k: np.concatenate([case[k], np.zeros(n, np.int32)]) for k in ("ctx", "qo", "qs", "ql")})
    pad["table"] = np.concatenate([case["table"], np.zeros((n, case["table"].shape[1]), np.int32)])
    assert _workspace(pkg, n + 2, 3, 3, 1, 64, 2, case["table"].shape[1], 64) == 0
    check_attention(pkg, dev, pad, f"ctx {ctx} unsplit")


@pytest.mark.parametrize("h_kv", [1, 2, 8])
def test_split_ranges(pkg, dev, h_kv):
    """Short chunks and decode rows of very different contexts in one split call, some with no key in later
    ranges, one without any; ranges and tiles that end together."""
    entries = [(20, 4076, 4096), (1, 9999, 10000), (3, 0, 3), (1, 1023, 1024), (33, 2100, 2133), (1, 4999, 5000),
               (5, 3000, 3005)]
    case = attention_case(50 + h_kv, entries, h=4 * h_kv, h_kv=h_kv, d=64, block_size=32)
    case["ctx"][6] = 0
    assert _workspace(pkg, 7, 64, 4 * h_kv, h_kv, 64, 33, case["table"].shape[1], 32) > 0
    o = check_attention(pkg, dev, case)
    assert not o[:, 59:64].any()
    # More entries than one wave looks at in a step, most of them empty.
    pad = {k: np.zeros((len(entries) + 60, *case[k].shape[1:]), np.int32) for k in ("table", "ctx", "qo", "qs", "ql")}
    at = np.arange(len(entries)) * 10 + 3
    for k in pad:
        pad[k][at] = case[k]
    if h_kv < 8:
        np.testing.assert_array_equal(attend(pkg, dev, dict(case, **pad)), o)
    else:
        check_attention(pkg, dev, dict(case, **pad))


def test_rows_of_no_entry_are_left_alone(pkg, dev):
    """Through the C entry point into a caller's o: rows before, between and behind the entries' keep what
    they held."""
    case = attention_case(36, [(3, 40, 43), (1, 1200, 1201), (2, 0, 2)], h=8, h_kv=2)
    want = attend(pkg, dev, case)
    q = np.zeros((8, 20, 128), np.uint16)
    at = [2, 3, 4, 9, 15, 16]
    q[:, at] = case["q"]
    qs = np.array([2, 9, 15], np.int32)
    pool = pool_to_dev(pkg, case["pool"], dev)
    qd = to_bf16_tensor(q, dev)
    o = torch.full((8, 20, 128), 7.0, dtype=torch.bfloat16, device=dev)
    table, ctx, qo, _, ql = attend_args(case, dev)
    nbytes = _workspace(pkg, 3, 20, 8, 2, 128, 3, table.shape[1], 16)
    ws = torch.full((max(nbytes, 16),), 0xff, dtype=torch.uint8, device=dev)  # NaN in what nobody writes
    start = i32(qs, dev)
    from llm_serving_engine_amd import _lib

    args = _lib.PAGED_ATTENTION_FP8_ARGS.pack(
        qd.data_ptr(), qd.stride(0), qd.stride(1), pool.k.data_ptr(), pool.v.data_ptr(), pool.k.stride(0),
        pool.scales.data_ptr(), pool.scales.stride(0), case["blocks"], 16, table.data_ptr(), table.stride(0),
        table.shape[1], ctx.data_ptr(), qo.data_ptr(), start.data_ptr(), ql.data_ptr(), o.data_ptr(),
        o.stride(0), o.stride(1), 3, 20, 3, 8, 2, 128, 128 ** -0.5)
    status = pkg.library().lse_paged_attention_fp8(args, ws.data_ptr(), nbytes,
                                                   torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status == 0
    np.testing.assert_array_equal(bf16_bits(o[:, at]), want)
    rest = [t for t in range(20) if t not in at]
    assert (o[:, rest] == 7.0).all()


def test_pool_past_32_bits(pkg, dev):
    """A pool of more than 4 GiB a side whose used blocks lie at its far end."""
    h_kv, d, bs = 8, 128, 64
    per, blocks = bs // 16, 70000
    case = attention_case(37, [(1, 199, 200), (70, 30, 100)], h=16, h_kv=h_kv, block_size=bs)
    want = attend(pkg, dev, case)
    own = case["pool"][0].shape[0]
    far = [torch.empty((blocks, h_kv, per, n), dtype=torch.uint8, device=dev) for n in (16 * d, 16 * d, 2)]
    assert far[0].numel() > 1 << 32
    for t, a in zip(far, case["pool"]):
        t[-own:] = torch.from_numpy(a).to(dev)
    pool = pkg.ops.Fp8KV(far[0].view(torch.float8_e4m3fn), far[1].view(torch.float8_e4m3fn),
                         far[2].view(torch.float8_e8m0fnu))
    table, *rest = attend_args(dict(case, table=case["table"] + blocks - own), dev)
    o = pkg.ops.paged_attention_fp8(to_bf16_tensor(case["q"], dev), pool, table, *rest, 70)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(bf16_bits(o), want)
    # The append at the same far end.
    rng = np.random.default_rng(37)
    x = to_dev(bf16_rows(rng, 71, h_kv, d), dev)
    plan = [i32(case[n], dev) for n in ("qo", "qs", "ql")]
    near = pool_to_dev(pkg, case["pool"], dev)
    pkg.ops.append_kv_fp8(None, x, x, None, None, near, i32(case["table"], dev), *plan, 70)
    pkg.ops.append_kv_fp8(None, x, x, None, None, pool, table, *plan, 70)
    for a, b in zip(pool, near):
        assert torch.equal(a.view(torch.uint8)[-own:], b.view(torch.uint8))


def test_strided_q_and_two_streams(pkg, dev):
    """q and k as slices of a stacked projection in token-major order, and two calls in flight at once."""
    case = attention_case(38, [(1, 5999, 6000), (3, 40, 43)], h=8, h_kv=2)
    want = attend(pkg, dev, case)
    stacked = torch.zeros(4, 12, 128, dtype=torch.bfloat16, device=dev)
    stacked[:, :8] = to_bf16_tensor(case["q"], dev).transpose(0, 1)
    pool, plan = pool_to_dev(pkg, case["pool"], dev), attend_args(case, dev)
    q = stacked[:, :8].transpose(0, 1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for stream in streams:
            with torch.cuda.stream(stream):
                got.append(pkg.ops.paged_attention_fp8(q, pool, *plan, 3))
    torch.cuda.synchronize()
    for o in got:
        assert o.shape == q.shape and o.stride(1) == 8 * 128  # token-major, as q
        np.testing.assert_array_equal(bf16_bits(o), want)


def test_attention_replays_from_a_graph(pkg, dev):
    """A split decode captured once, replayed over growing contexts with eager calls between; two graphs."""
    case = attention_case(39, [(1, 1500, 1501), (1, 30, 31)], h=8, h_kv=2)
    case["table"] = np.concatenate([case["table"], np.zeros_like(case["table"][:, :1])], 1)
    pool = pool_to_dev(pkg, case["pool"], dev)
    q = to_bf16_tensor(case["q"], dev)
    table, ctx, qo, qs, ql = attend_args(case, dev)
    call = lambda: pkg.ops.paged_attention_fp8(q, pool, table, ctx, qo, qs, ql, 1)  # noqa: E731
    call()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for step in range(3):
        for g, o in zip(graphs, outs):
            q.mul_(-1.25)
            g.replay()
            want = call()
            torch.cuda.synchronize()
            assert torch.equal(o, want)
        ctx.add_(1)
        qo.add_(1)


def test_append_then_attend(pkg, dev):
    """The operators as a serving loop uses them: prompts appended in chunks beside decoding sequences, then
    decode steps, each step's rows attended; against fp64 attention over the unpacked cache, and that cache
    against the rotated rows within its codes' rounding."""
    rng = np.random.default_rng(40)
    h, h_kv, d, bs, rotary = 8, 2, 128, 32, 64
    cos, sin = pkg.ops.rope_table(512, rotary, 10000.0, device=dev)
    pool = pkg.ops.fp8_kv_pool(40, bs, h_kv, d, dev)
    table = rng.permutation(40)[:36].reshape(3, 12).astype(np.int32)
    lens = [0, 0, 0]
    kept = [[], [], []]
    for step in [(70, 0, 1), (50, 33, 1), (1, 64, 1), (1, 1, 1), (1, 1, 0), (1, 1, 17)]:
        ql = np.array(step, np.int32)
        tokens = int(ql.sum())
        x = bf16_rows(rng, tokens, h + 2 * h_kv, d)
        qkv = to_dev(x, dev)
        plan = dict(qo=np.array(lens, np.int32), ql=ql, ctx=np.array(lens, np.int32) + ql, table=table,
                    qs=np.concatenate([[0], np.cumsum(ql)[:-1]]).astype(np.int32))
        qo, qs, qlen, ctx, tab = (i32(plan[n], dev) for n in ("qo", "qs", "ql", "ctx", "table"))
        most = int(ql.max())
        q = pkg.ops.append_kv_fp8(qkv[:, :h], qkv[:, h:h + h_kv], qkv[:, h + h_kv:], cos, sin, pool, tab, qo,
                                  qs, qlen, most, interleaved=True)
        o = pkg.ops.paged_attention_fp8(q.transpose(0, 1), pool, tab, ctx, qo, qs, qlen, most)
        torch.cuda.synchronize()
        pos = np.concatenate([np.arange(a, a + n) for a, n in zip(lens, ql)]).astype(np.int64)
        c, s = cos.cpu().numpy(), sin.cpu().numpy()
        krot = kv.rotate(x[:, h:h + h_kv], c, s, pos, True)
        host = tuple(t.view(torch.uint8).cpu().numpy() for t in pool)
        golden, covered, vmax = attention_golden(dict(plan, q=bf16_bits(q.transpose(0, 1)), pool=host, bs=bs))
        ok, msg = ora.attention_within_tolerance(bf16_bits(o), golden, vmax, covered)
        assert ok, msg
        for e, n in enumerate(ql):
            rows = slice(int(plan["qs"][e]), int(plan["qs"][e]) + int(n))
            kept[e] += list(krot[rows])
            lens[e] += int(n)
        values, _ = kv.unpack(host, bs)
        for e in range(3):
            for p in range(lens[e]):
                block, sub = table[e, p // bs], p % bs // 16
                scale = 2.0 ** (host[2][block, :, sub, 0].astype(np.int64) - 127)[:, None]
                want = kept[e][p].astype(np.float64)
                assert (np.abs(values[block, p % bs] - want)
                        <= 2.0 ** -4 * np.abs(want) + 2.0 ** -9 * scale).all()


SOURCES = Path(__file__).resolve().parent.parent / "llm-serving-engine_amd" / "csrc"


def _tiled(case, most=None):
    """Whether the row-tiled kernel takes the case's long entries (128 rows per K/V head), by the library's own
    bounds."""
    text = (SOURCES / "attn_fp8.hip").read_text() + (SOURCES / "attn_fp8.h").read_text()
    bound = {n: float(v) for n, v in re.findall(r"\bk(\w+) = ([\d.e]+)[,;]", text)}
    h, tokens, _ = case["q"].shape
    h_kv, entries = case["pool"][0].shape[1], len(case["ql"])
    g, most = h // h_kv, most or int(case["ql"].max())
    if most * g < bound["F8LongRows"]:
        return False
    q, rows = min(most, tokens), tokens * g
    left = rows if rows >= entries * bound["F8LongRows"] else rows - entries * (bound["F8LongRows"] - 1)
    room = case["table"].shape[1] * case["bs"]
    enough = bound["Items256" if room <= 256 else "Items512" if room <= 512 else "Items"]
    if max(-(-q * g // 128), left // 128) * h_kv >= enough:
        return True
    keys = max(room - q // 2, 0)
    pairs = rows * h_kv * keys * (1 if keys < bound["Far"] else 2)
    return pairs >= (bound["PairsMixed"] if (entries - 1) * h_kv >= bound["Mixed"] else bound["Pairs"])


def _long_case(*args, **kw):
    case = attention_case(*args, **kw)
    assert _tiled(case)
    return case


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,h_kv", [(80, 20), (99, 33), (240, 15), (105, 105)])
def test_long_entries(pkg, dev, h, h_kv, d):
    """Entries on both sides of the first row-tiled length and of the next row tile, key tiles one short of and
    one over, decode rows beside them."""
    g = h // h_kv
    first = -(-128 // g)
    entries = [(first - 1, 5, first + 4), (first, 0, first), (first + 1, 700, first + 701),
               (384 // g, 63, 384 // g + 63), (384 // g + 1, 64, 384 // g + 65), (1, 600, 601), (1, 0, 1),
               (640 // g, 0, 640 // g)]
    check_attention(pkg, dev, _long_case(h + d, entries, h=h, h_kv=h_kv, d=d, block_size=48), f"{h} over {h_kv}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("entries", [[(300, 17000, 17300)], [(300, 19000, 19300), (1, 18000, 18001), (40, 70, 110)]])
def test_parts_of_few_items(pkg, dev, entries, d):
    """Few items behind long contexts are cut into 16 parts by their keys; beside a decode row whose keys are
    split too, and a long entry that has one part."""
    case = _long_case(70 + len(entries), entries, h=4, h_kv=1, d=d, block_size=64)
    check_attention(pkg, dev, case, "parts")


@pytest.mark.parametrize("entries,h,h_kv,d,tiled", [
    ([(64, 0, 64)] * 5, 32, 8, 64, True), ([(64, 0, 64)] * 4, 32, 8, 64, False),
    ([(64, 300, 364)] * 8, 32, 8, 64, True), ([(64, 300, 364)] * 7, 32, 8, 64, False)])
def test_short_prompts_on_both_sides_of_the_rule(pkg, dev, entries, h, h_kv, d, tiled):
    case = attention_case(69, entries, h=h, h_kv=h_kv, d=d)
    assert _tiled(case) == tiled
    check_attention(pkg, dev, case, f"{len(entries)} prompts")


@pytest.mark.parametrize("end", [1, 63, 64, 65, 127, 128, 129, 191, 192, 193, 385, 500])
def test_long_entries_key_edges(pkg, dev, end):
    """Contexts one short of and one over a key tile; the second entry's rows see less and less, the third's
    nothing."""
    case = _long_case(end, [(64, max(end - 64, 0), max(end, 64)), (70, 11, 81), (64, 0, 64)], h=136, h_kv=34, d=64)
    case["ctx"][:] = [end, min(end, 81), 0]
    o = check_attention(pkg, dev, case, f"end {end}")
    assert not o[:, 134:].any()


@pytest.mark.parametrize("q_scale", [0.0, 3.0, 2.0 ** 12, 2.0 ** 40, 2.0 ** -40])
def test_long_entries_flat_and_peaked_scores(pkg, dev, q_scale):
    case = _long_case(61, [(150, 450, 600), (64, 0, 64)], h=136, h_kv=34, q_scale=q_scale)
    check_attention(pkg, dev, case, f"q x {q_scale}")


def test_long_entries_read_nothing_behind_their_context(pkg, dev):
    """NaN codes in every slot behind a context, NaN scales in groups behind it, a bad block in one entry."""
    entries = [(80, 20, 100), (64, 300, 364), (70, 0, 70), (1, 40, 41)]
    case = _long_case(62, entries, h=136, h_kv=34, d=128, block_size=16)
    want = attend(pkg, dev, case)
    k, v, s = (a.copy() for a in case["pool"])
    used = np.zeros((case["blocks"], 16), bool)
    for e, (_, _, ctx) in enumerate(entries):
        for n in range(ctx):
            used[case["table"][e, n // 16], n % 16] = True
    dims = np.arange(128)
    for b, slot in np.argwhere(~used):
        k[b, :, 0, kv.k_index(slot, dims, 128)] = 127
        v[b, :, 0, kv.v_index(slot, dims, 128)] = 255
        if not used[b].any():
            s[b] = kv.NAN_SCALE
    case["pool"] = (k, v, s)
    np.testing.assert_array_equal(attend(pkg, dev, case), want)
    case["table"] = case["table"].copy()
    case["table"][1, 3] = case["blocks"] + 5
    o = ora.bf16_bits_to_f32(attend(pkg, dev, case))
    assert np.isnan(o[:, 80:144]).all()
    np.testing.assert_array_equal(ora.f32_to_bf16_bits(o[:, :80]), want[:, :80])
    np.testing.assert_array_equal(ora.f32_to_bf16_bits(o[:, 144:]), want[:, 144:])


@pytest.mark.parametrize("h,h_kv,tiled", [(16, 1, True), (4, 1, True), (2, 1, False)])
def test_many_entries(pkg, dev, h, h_kv, tiled):
    """More entries than a wave looks at in a step: prompts of 64 to 100 tokens among decode rows."""
    rng = np.random.default_rng(63)
    entries = [(int(n), int(o), int(n + o)) for n, o in zip(rng.integers(64, 100, 70), rng.integers(0, 90, 70))]
    entries = [x for e in entries for x in (e, (1, e[2], e[2] + 1))]
    case = attention_case(63, entries, h=h, h_kv=h_kv, d=64)
    assert _tiled(case) == tiled
    check_attention(pkg, dev, case, "many")


def test_long_entries_replay_from_a_graph(pkg, dev):
    """A mixed call whose items are cut into parts, captured once, replayed with other q, against eager calls."""
    case = _long_case(64, [(300, 17000, 17300), (1, 3000, 3001), (2, 7, 9)], h=4, h_kv=1, d=64, block_size=64)
    pool, q, plan = pool_to_dev(pkg, case["pool"], dev), to_bf16_tensor(case["q"], dev), attend_args(case, dev)
    call = lambda: pkg.ops.paged_attention_fp8(q, pool, *plan, 300)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call()
    for _ in range(3):
        q.mul_(-1.25)
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(o, want)


def test_how_far_a_nan_value_reaches(pkg, dev):
    """NaN in a token's v: the rows that see it, and earlier rows of its own query tile at most (16 query rows, or
    128 of a long entry); no other entry or K/V head."""
    for h, h_kv, reach in ((8, 2, 16), (128, 32, 128)):
        case = attention_case(65, [(150, 0, 150), (150, 0, 150)], h=h, h_kv=h_kv, d=64)
        assert _tiled(case) == (reach == 128)
        want = attend(pkg, dev, case)
        v = case["pool"][1].copy()
        v[case["table"][0, 120 // 16], 1, 0, kv.v_index(120 % 16, np.arange(64), 64)] = 127
        o = attend(pkg, dev, dict(case, pool=(case["pool"][0], v, case["pool"][2])))
        nan = np.isnan(ora.bf16_bits_to_f32(o)).any(-1)
        g = h // h_kv
        assert nan[g:2 * g, 120:150].all()
        assert not nan[:, 150:].any() and not nan[:g].any() and not nan[2 * g:].any()
        assert not nan[:, :max(0, 120 - reach // g + 1)].any()
        np.testing.assert_array_equal(o[~nan], want[~nan])
