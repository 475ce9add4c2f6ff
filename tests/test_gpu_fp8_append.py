"""Rotary positions and the append into the 8-bit paged K/V cache on the GPU against the fp64 / element-by-
element restatement. Codes and scales have one right value and are compared byte for byte; rotated rows are
rounded once, to bf16."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fp8_kv_helpers import (bf16_rows, i32, plan_of, pool_to_dev, pool_to_host, random_pool, same_pool,
                            to_dev)
from helpers import bf16_bits
from oracle import kv_cache as kv
from oracle import numerics as ora

pytestmark = pytest.mark.gpu

THETA = 10000.0


def _tables(pkg, dev, rows, rotary):
    cos, sin = pkg.ops.rope_table(rows, rotary, THETA, device=dev)
    return cos, sin, cos.cpu().numpy(), sin.cpu().numpy()


def _check_rotated(got, x, cos, sin, positions, interleaved):
    """bf16 rows within half a step (2^-8 of the value) and the three fp32 roundings (each 2^-24 of at most
    |a c| + |b s|) of the fp64 rotation; dims behind the rotated ones bit for bit."""
    exact = kv.rotate(x, cos, sin, positions, interleaved, np.float64)
    size = kv.rotate(np.abs(x), np.abs(cos), -np.abs(sin), positions, interleaved, np.float64)
    size = np.maximum(size, kv.rotate(np.abs(x), np.abs(cos), np.abs(sin), positions, interleaved, np.float64))
    y = ora.bf16_bits_to_f32(bf16_bits(got)).astype(np.float64)
    assert (np.abs(y - exact) <= 2.0 ** -8 * np.abs(exact) + 2.0 ** -21 * np.abs(size) + 1e-38).all()
    np.testing.assert_array_equal(y[..., 2 * cos.shape[1]:], x[..., 2 * cos.shape[1]:])
    # The same in fp32 operations, which the kernel's are: no difference at all.
    want = ora.f32_to_bf16_bits(kv.rotate(x, cos, sin, positions, interleaved).astype(np.float32))
    np.testing.assert_array_equal(bf16_bits(got), want)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,h,h_kv,d,rotary", [
    (1, 32, 8, 128, 128), (7, 24, 8, 128, 64), (33, 5, 1, 64, 32), (257, 3, 3, 80, 32), (2, 2, 2, 16, 16),
    (5, 1, 1, 1024, 1024), (64, 8, 2, 96, 48)])
def test_rope(pkg, dev, tokens, h, h_kv, d, rotary, interleaved):
    rng = np.random.default_rng(tokens + d)
    cos, sin, c, s = _tables(pkg, dev, 700, rotary)
    pos = rng.integers(0, 700, tokens)
    q, k = bf16_rows(rng, tokens, h, d), bf16_rows(rng, tokens, h_kv, d, scale=30.0)
    got = pkg.ops.rope(to_dev(q, dev), to_dev(k, dev), cos, sin, i32(pos, dev), interleaved=interleaved)
    for y, x in zip(got, (q, k)):
        assert y.shape == x.shape and y.is_contiguous()
        _check_rotated(y, x, c, s, pos, interleaved)


def test_rope_strides_and_no_k(pkg, dev):
    """q and k as slices of a stacked projection, head-major q, an address off 16 bytes, q alone."""
    rng = np.random.default_rng(1)
    cos, sin, c, s = _tables(pkg, dev, 50, 64)
    pos = rng.integers(0, 50, 9)
    x = bf16_rows(rng, 9, 10, 64)
    stacked = to_dev(x, dev)
    q, k = pkg.ops.rope(stacked[:, :6], stacked[:, 6:8], cos, sin, i32(pos, dev))
    _check_rotated(q, x[:, :6], c, s, pos, False)
    _check_rotated(k, x[:, 6:8], c, s, pos, False)
    heads = stacked.transpose(0, 1).contiguous().transpose(0, 1)
    q, none = pkg.ops.rope(heads, None, cos, sin, i32(pos, dev))
    assert none is None
    _check_rotated(q, x, c, s, pos, False)
    flat = torch.empty(9 * 640 + 1, dtype=torch.bfloat16, device=dev)
    odd = flat[1:].view(9, 10, 64)
    odd.copy_(stacked)
    _check_rotated(pkg.ops.rope(odd, None, cos, sin, i32(pos, dev))[0], x, c, s, pos, False)
    empty = pkg.ops.rope(stacked[:0], stacked[:0], cos, sin, i32(pos[:0], dev))
    assert empty[0].shape == (0, 10, 64)


def test_rope_positions_outside_the_tables(pkg, dev):
    rng = np.random.default_rng(2)
    cos, sin, c, s = _tables(pkg, dev, 20, 32)
    x = bf16_rows(rng, 4, 2, 64)
    got, _ = pkg.ops.rope(to_dev(x, dev), None, cos, sin, i32([3, 20, -1, 19], dev))
    _check_rotated(got[[0, 3]], x[[0, 3]], c, s, np.array([3, 19]), False)
    y = got.float().cpu().numpy()
    assert np.isnan(y[1:3, :, :32]).all()
    np.testing.assert_array_equal(y[1:3, :, 32:], x[1:3, :, 32:])


def _append_case(seed, news, h=8, h_kv=2, d=64, block_size=16, scale=1.0, spare=2):
    """news: (new tokens, positions before them)."""
    rng = np.random.default_rng(seed)
    case = plan_of(rng, [(n, o, n + o) for n, o in news], block_size, spare)
    tokens = int(case["ql"].sum())
    case.update(q=bf16_rows(rng, tokens, h, d), k=bf16_rows(rng, tokens, h_kv, d, scale=scale),
                v=bf16_rows(rng, tokens, h_kv, d, scale=scale), bs=block_size,
                pool=random_pool(rng, case["blocks"], block_size, h_kv, d))
    return case


def _append(pkg, dev, case, cos, sin, interleaved=False, pool=None, q=True, most=None):
    pool = pool or pool_to_dev(pkg, case["pool"], dev)
    plan = [i32(case[n], dev) for n in ("table", "qo", "qs", "ql")]
    got = pkg.ops.append_kv_fp8(to_dev(case["q"], dev) if q else None, to_dev(case["k"], dev),
                                to_dev(case["v"], dev), cos, sin, pool, *plan,
                                most or int(case["ql"].max()), interleaved=interleaved)
    torch.cuda.synchronize()
    return got, pool


def _positions(case):
    return np.concatenate([np.arange(o, o + n) for n, o in zip(case["ql"], case["qo"])]).astype(np.int64)


def _want(case, c, s, interleaved=False, pool=None):
    k = case["k"] if c is None else kv.rotate(case["k"], c, s, _positions(case), interleaved)
    pool = tuple(a.copy() for a in (pool or case["pool"]))
    kv.append(pool, k, case["v"], case["table"], case["qo"], case["qs"], case["ql"], case["bs"])
    return pool


RAGGED = [(1, 0), (1, 15), (1, 16), (0, 5), (17, 0), (16, 32), (15, 1), (2, 30), (40, 7), (1, 200), (33, 15)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,h,h_kv,rotary,block_size", [
    (64, 8, 2, 64, 16), (64, 3, 3, 16, 48), (128, 24, 8, 128, 16), (128, 16, 1, 32, 64), (128, 10, 2, 64, 32)])
def test_append_ragged(pkg, dev, d, h, h_kv, rotary, block_size, interleaved):
    """New tokens that start and end anywhere in a group, empty entries among them."""
    cos, sin, c, s = _tables(pkg, dev, 300, rotary)
    case = _append_case(d + h, RAGGED, h, h_kv, d, block_size)
    q, pool = _append(pkg, dev, case, cos, sin, interleaved)
    same_pool(pool_to_host(pool), _want(case, c, s, interleaved))
    _check_rotated(q, case["q"], c, s, _positions(case), interleaved)


@pytest.mark.parametrize("entries", [1, 63, 64, 65, 130])
def test_append_decode_batches(pkg, dev, entries):
    """One token of each sequence (the direct grid), and with one longer entry (the counted one)."""
    cos, sin, c, s = _tables(pkg, dev, 200, 64)
    rng = np.random.default_rng(entries)
    news = [(1, int(o)) for o in rng.integers(0, 150, entries)]
    for extra in ([], [(37, 3)]):
        case = _append_case(entries, news + extra)
        q, pool = _append(pkg, dev, case, cos, sin)
        same_pool(pool_to_host(pool), _want(case, c, s))
        _check_rotated(q, case["q"], c, s, _positions(case), False)


def test_append_without_q_or_rotation(pkg, dev):
    case = _append_case(5, RAGGED)
    q, pool = _append(pkg, dev, case, None, None, q=False)
    assert q is None
    same_pool(pool_to_host(pool), _want(case, None, None))
    q, pool = _append(pkg, dev, case, None, None)
    np.testing.assert_array_equal(q.float().cpu().numpy(), case["q"])
    same_pool(pool_to_host(pool), _want(case, None, None))


@pytest.mark.parametrize("steps", [[1] * 40, [5, 1, 20, 3, 16, 1, 1]])
def test_a_sequence_appended_in_pieces(pkg, dev, steps):
    """Token by token and chunk by chunk with rows that grow: every step requantises the half-filled group.
    Against the same steps restated, and against the values: a code is off by half a step of its scale
    (2^-4 of the value, 2^-10 of the scale below 2^-6 of it), a requantised one once more below there."""
    rng = np.random.default_rng(len(steps))
    pool = pool_np = None
    rows_k = []
    for i, n in enumerate(steps):
        case = _append_case(100 + i, [(n, sum(steps[:i]))], block_size=16)
        case["table"] = np.arange(5, dtype=np.int32)[None]
        case["k"] = bf16_rows(rng, n, 2, 64, scale=2.0 ** (i % 9 - 4))
        rows_k.append(case["k"])
        case["pool"] = pool_np or random_pool(rng, 5, 16, 2, 64)
        _, pool = _append(pkg, dev, case, None, None, pool=pool)
        pool_np = _want(case, None, None)
        same_pool(pool_to_host(pool), pool_np)
    got = pkg.ops.unpack_fp8_kv(pool)[0].double().cpu().numpy().reshape(80, 2, 64)
    for p, x in enumerate(np.concatenate(rows_k).astype(np.float64)):
        scale = 2.0 ** (pool_np[2][p // 16, :, 0, 0].astype(np.int64) - 127)[:, None]
        assert (np.abs(got[p] - x) <= 2.0 ** -4 * np.abs(x) + 2 * 2.0 ** -10 * scale).all()


def test_extreme_rows(pkg, dev):
    """Zeros, the largest and the least bf16 values, infinities and NaN (held as NaN, out of the scale), a
    group whose former scale is NaN."""
    case = _append_case(7, [(16, 0), (16, 16), (16, 0), (16, 0), (4, 8), (3, 9)], h=2, h_kv=2, d=64)
    big = float(torch.finfo(torch.bfloat16).max)
    case["k"][:16], case["v"][:16] = 0.0, -0.0
    case["k"][16:32] *= big / np.abs(case["k"][16:32]).max() * 0.99
    case["v"][16:32, :, 0] = big
    case["k"][32:48] *= 2.0 ** -130
    case["v"][32:48] *= 2.0 ** -126
    case["k"][48, 0, 3], case["k"][50, 0, 7], case["v"][51, 1, 0] = np.inf, np.nan, -np.inf
    case["v"][52] = np.nan
    for name in ("k", "v"):
        case[name] = ora.bf16_bits_to_f32(ora.f32_to_bf16_bits(case[name].astype(np.float32)))
    case["pool"][2][case["table"][4, 0], :, 0] = kv.NAN_SCALE
    case["pool"][2][case["table"][5, 0], :, 0] = 254
    _, pool = _append(pkg, dev, case, None, None)
    same_pool(pool_to_host(pool), _want(case, None, None))


def test_what_is_dropped_and_what_stays(pkg, dev):
    """Blocks outside the pool, positions past the table, negative offsets, rows outside the call's: nothing
    of them is written, and no byte of other groups changes. Their q rows are rotated all the same."""
    case = _append_case(9, [(20, 0), (20, 30), (5, 3), (4, 20), (3, 0)])
    case["table"][0, 1] = case["blocks"]
    case["table"][2, 0] = -1
    case["table"] = np.ascontiguousarray(case["table"][:, :2])  # entry 1's positions from 32 on, entry 3's last
    case["qo"][4] = -2
    case["qs"][3] = 50  # rows 50 and 51 are entry 4's, the others outside
    cos, sin, c, s = _tables(pkg, dev, 64, 64)
    q, pool = _append(pkg, dev, case, None, None)
    same_pool(pool_to_host(pool), _want(case, None, None))


@pytest.mark.parametrize("start", [150, 90, -70, -300])
def test_rows_outside_take_no_other_entrys_place(pkg, dev, start):
    """An entry of many rows outside the call's, before entries whose rows all lie inside."""
    case = _append_case(10, [(100, 7), (5, 40), (60, 3), (1, 0)])
    case["qs"][0] = start
    q, pool = _append(pkg, dev, case, None, None)
    same_pool(pool_to_host(pool), _want(case, None, None))


def test_padding_rows_and_entries(pkg, dev):
    """A graph bucket: entries of no tokens behind the real ones, rows of no entry, a table as wide as the
    pool, a larger max_q_len."""
    case = _append_case(11, RAGGED)
    want = _want(case, None, None)
    e = len(RAGGED)
    wide = np.full((e + 9, case["blocks"]), case["blocks"] - 1, np.int32)
    wide[:e, :case["table"].shape[1]] = case["table"]
    pad = dict(case, table=wide, **{n: np.concatenate([case[n], np.zeros(9, np.int32)]) for n in ("qo", "qs", "ql")})
    for name in ("q", "k", "v"):
        pad[name] = np.concatenate([case[name], np.full_like(case[name][:7], np.nan)])
    q, pool = _append(pkg, dev, pad, None, None, most=64)
    same_pool(pool_to_host(pool), want)


def test_pool_blocks_may_be_strided(pkg, dev):
    """k and v of one allocation, block by block; and pools whose blocks lie far apart."""
    case = _append_case(13, RAGGED, block_size=32)
    want = _want(case, None, None)
    k, v, sc = pool_to_dev(pkg, case["pool"], dev)
    both = torch.stack([k.view(torch.uint8), v.view(torch.uint8)], 1).view(torch.float8_e4m3fn)
    wide = torch.zeros(2 * len(sc), *sc.shape[1:], dtype=torch.uint8, device=dev)
    wide[::2] = sc.view(torch.uint8)
    pool = pkg.ops.Fp8KV(both[:, 0], both[:, 1], wide.view(torch.float8_e8m0fnu)[::2])
    _append(pkg, dev, case, None, None, pool=pool)
    same_pool(pool_to_host(pool), want)


def test_append_replays_from_a_graph(pkg, dev):
    """Captured once, replayed over changed rows and offsets with eager calls between."""
    case = _append_case(15, [(1, 5), (1, 31), (1, 100)])
    pool, eager_pool = (pool_to_dev(pkg, case["pool"], dev) for _ in range(2))
    cos, sin, c, s = _tables(pkg, dev, 300, 64)
    x = {n: to_dev(case[n], dev) for n in ("q", "k", "v")}
    table, qo, qs, ql = (i32(case[n], dev) for n in ("table", "qo", "qs", "ql"))
    table = torch.cat([table, torch.zeros_like(table[:, :1])], 1)
    call = lambda p: pkg.ops.append_kv_fp8(x["q"], x["k"], x["v"], cos, sin, p, table, qo, qs, ql, 1)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        scratch = pool_to_dev(pkg, case["pool"], dev)
        call(scratch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(pool)
    for step in range(4):
        x["k"].mul_(-1.5)
        qo.add_(1 if step else 0)
        graph.replay()
        want = call(eager_pool)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        same_pool(pool_to_host(pool), pool_to_host(eager_pool))
