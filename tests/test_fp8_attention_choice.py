"""Which kernel a call of the 8-bit cache's attention runs, and into how many parts and ranges it cuts its work, as the
library itself tells: literal sizes on both sides of every bound; no GPU."""

from __future__ import annotations

import ctypes

import pytest

from fp8_attention_helpers import choice, pack


@pytest.mark.parametrize("entries,tokens,most,h,h_kv,room,tiled", [
    # An entry of 128 query rows per K/V head, 32 tokens of 4 heads each, is the shortest that it takes.
    (9, 9 * 31, 31, 32, 8, 32, False), (9, 9 * 32, 32, 32, 8, 32, True), (9, 9 * 7, 7, 128, 8, 32, False),
    (9, 9 * 8, 8, 128, 8, 32, True), (20, 20 * 127, 127, 8, 8, 128, False), (20, 20 * 128, 128, 8, 8, 128, True),
    # 72 items of 128 rows behind up to 256 positions, 128 behind up to 512, 200 behind more.
    (8, 8 * 32, 32, 32, 8, 256, False), (9, 9 * 32, 32, 32, 8, 256, True), (9, 9 * 32, 32, 32, 8, 272, False),
    (15, 15 * 32, 32, 32, 8, 512, False), (16, 16 * 32, 32, 32, 8, 512, True), (12, 12 * 64, 64, 32, 8, 528, False),
    (13, 13 * 64, 64, 32, 8, 528, True), (1, 768, 768, 32, 8, 1024, False), (1, 800, 800, 32, 8, 1024, True),
    # 40 million (query row, key) pairs, which count twice from 6000 positions on.
    (1, 512, 512, 32, 8, 2688, False), (1, 512, 512, 32, 8, 2704, True), (1, 128, 128, 32, 8, 6048, False),
    (1, 128, 128, 32, 8, 6064, True),
    # 12 million beside entries that fill half the card: 16 others of 8 K/V heads.
    (17, 144, 128, 32, 8, 2656, False), (17, 144, 128, 32, 8, 2672, True), (16, 143, 128, 32, 8, 2672, False),
    # Decode rows alone never.
    (512, 512, 1, 32, 8, 1 << 20, False)])
def test_which_kernel(pkg, entries, tokens, most, h, h_kv, room, tiled):
    for d in (64, 128):
        got = choice(pkg, entries, tokens, most, h, h_kv, d, room)
        assert got[0] == tiled and (got[1] > 0) == tiled


@pytest.mark.parametrize("entries,tokens,most,h,h_kv,room,parts", [
    (1, 420, 420, 16, 4, 6512, 9),        # 14 items of 4 heads: 512 / 56
    (1, 300, 300, 4, 1, 17408, 16),       # as many as there are, at most
    (1, 600, 600, 32, 8, 2512, 3),        # 152 items
    (1, 1813, 1813, 32, 8, 8080, 1),      # 456 items: whole ones
    (41, 340, 300, 24, 8, 2000, 3),       # 64 items beside 320 decoding: 512 / 144
    (41, 440, 400, 32, 8, 1312, 2),       # 104 beside 320: 512 / 184
    (41, 440, 400, 32, 8, 1136, 2), (41, 885, 845, 24, 8, 2832, 2), (9, 9 * 32, 32, 32, 8, 256, 1)])
def test_parts(pkg, entries, tokens, most, h, h_kv, room, parts):
    got = choice(pkg, entries, tokens, most, h, h_kv, 128, room)
    assert got[:2] == (True, parts)


@pytest.mark.parametrize("entries,tokens,most,h,h_kv,room,units", [
    (63, 63, 1, 32, 8, 2064, 64), (64, 64, 1, 32, 8, 2064, 0), (63, 63, 1, 32, 8, 2048, 0), (1, 1, 1, 32, 8, 2064, 64),
    (7, 64, 33, 8, 2, 10016, 256), (1, 1, 1, 16, 1, 1 << 20, 512), (1, 2, 2, 600, 600, 4096, 0),
    (1, 1813, 1813, 32, 8, 8080, 0)])  # a lone long entry: nothing is left to split
def test_split_keys(pkg, entries, tokens, most, h, h_kv, room, units):
    assert choice(pkg, entries, tokens, most, h, h_kv, 128, room)[2] == units


def test_workspaces_agree_with_the_choice(pkg):
    """Partial states are what a workspace holds: none without parts or split keys."""
    lib = pkg.library()
    for entries, tokens, most, room in [(1, 1, 1, 2048), (1, 1, 1, 4096), (64, 64, 1, 4096), (41, 440, 400, 1312),
                                        (1, 1813, 1813, 8080), (1, 600, 600, 2512), (9, 288, 32, 256)]:
        tiled, parts, units = choice(pkg, entries, tokens, most, 32, 8, 128, room)
        size = lib.lse_paged_attention_fp8_workspace_bytes(pack(
            block_size=16, max_blocks=room // 16, entries=entries, tokens=tokens, most=most, h=32, h_kv=8, d=128))
        assert (size > 0) == (parts > 1 or units > 0)


def test_refusals(pkg):
    lib = pkg.library()
    v = [ctypes.c_int64(-1) for _ in range(3)]
    out = [ctypes.byref(x) for x in v]
    good = dict(block_size=16, max_blocks=4, entries=1, tokens=1, most=1, h=8, h_kv=2, d=64)
    assert lib.lse_paged_attention_fp8_choice(None, *out) == -1
    assert lib.lse_paged_attention_fp8_choice(pack(**good), out[0], None, out[2]) == -1
    assert lib.lse_paged_attention_fp8_choice(pack(**{**good, "d": 96}), *out) == -2
    assert lib.lse_paged_attention_fp8_choice(pack(**{**good, "max_blocks": 1 << 27}), *out) == -4
    assert [x.value for x in v] == [-1] * 3
    assert lib.lse_paged_attention_fp8_choice(pack(**{**good, "entries": 0}), *out) == 0
    assert [x.value for x in v] == [0] * 3
