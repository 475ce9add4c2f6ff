"""Refusals of the 8-bit cache's entry points, without a GPU: every call below is turned down before any HIP
call is made."""

from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

FAKE = 1 << 20  # a 256-byte-aligned device address that is never used
E_NULL, E_SHAPE, E_ALIGN, E_RANGE, E_WORKSPACE = -1, -2, -3, -4, -6

ROPE = dict(q=FAKE, q_t=512, q_h=64, k=FAKE, k_t=128, k_h=64, cos=FAKE, sin=FAKE, rows=100, positions=FAKE,
            q_out=FAKE, k_out=FAKE, tokens=4, h=8, h_kv=2, d=64, rotary=64, interleaved=0)
APPEND = dict(q=FAKE, q_t=512, q_h=64, k=FAKE, k_t=128, k_h=64, v=FAKE, v_t=128, v_h=64, cos=FAKE, sin=FAKE,
              rows=100, q_out=FAKE, k_pool=FAKE, v_pool=FAKE, stride=2048, scales=FAKE, s_stride=4, blocks=10,
              block_size=16, table=FAKE, t_stride=5, max_blocks=5, offset=FAKE, start=FAKE, length=FAKE,
              entries=3, tokens=4, most=2, h=8, h_kv=2, d=64, rotary=64, interleaved=0)
ATTEND = dict(q=FAKE, q_h=256, q_t=64, k_pool=FAKE, v_pool=FAKE, stride=2048, scales=FAKE, s_stride=4,
              blocks=10, block_size=16, table=FAKE, t_stride=5, max_blocks=5, ctx=FAKE, offset=FAKE, start=FAKE,
              length=FAKE, o=FAKE, o_h=256, o_t=64, entries=3, tokens=4, most=2, h=8, h_kv=2, d=64,
              scale=0.125)


def _pack(pkg, layout, base, changes):
    """The packed argument struct: null pointers are 0."""
    assert set(changes) <= set(base)
    return layout.pack(*(0 if v is None else v for v in {**base, **changes}.values()))


def _call(pkg, name, base, changes):
    from llm_serving_engine_amd import _lib

    layout = dict(lse_rope=_lib.ROPE_ARGS, lse_append_kv_fp8=_lib.APPEND_KV_FP8_ARGS)[name]
    return getattr(pkg.library(), name)(_pack(pkg, layout, base, changes), None)


def _attend(pkg, changes, ws=None, ws_bytes=0):
    from llm_serving_engine_amd import _lib

    args = _pack(pkg, _lib.PAGED_ATTENTION_FP8_ARGS, ATTEND, changes)
    return pkg.library().lse_paged_attention_fp8(args, ws, ws_bytes, None)


def test_the_structs_are_the_headers(pkg):
    """As many fields as the header's structs have, each of eight bytes."""
    from llm_serving_engine_amd import _lib

    text = (Path(__file__).resolve().parent.parent / "include" / "lse_int8.h").read_text()
    for name, layout, base in (("lse_rope_args", _lib.ROPE_ARGS, ROPE),
                               ("lse_append_kv_fp8_args", _lib.APPEND_KV_FP8_ARGS, APPEND),
                               ("lse_paged_attention_fp8_args", _lib.PAGED_ATTENTION_FP8_ARGS, ATTEND)):
        body = re.search(r"struct " + name + r" \{(.*?)\};", text, re.S).group(1)
        fields = 0
        for line in body.split(";"):
            line = line.strip()
            if line:
                assert re.match(r"(const )?(void|float|int32_t)( ?\*)|int64_t |double ", line), line
                fields += line.count(",") + 1
        assert layout.size == 8 * fields == 8 * len(base)


def test_no_arguments_at_all(pkg):
    lib = pkg.library()
    assert lib.lse_rope(None, None) == lib.lse_append_kv_fp8(None, None) == E_NULL
    assert lib.lse_paged_attention_fp8(None, None, 0, None) == E_NULL
    assert lib.lse_paged_attention_fp8_workspace_bytes(None) == -1


@pytest.mark.parametrize("changes,status", [
    (dict(d=72), E_SHAPE), (dict(d=1040), E_SHAPE), (dict(rotary=8), E_SHAPE), (dict(rotary=80), E_SHAPE),
    (dict(rotary=24), E_SHAPE), (dict(tokens=-1), E_SHAPE), (dict(h=0), E_SHAPE), (dict(rows=0), E_SHAPE),
    (dict(interleaved=2), E_SHAPE), (dict(q=None), E_NULL), (dict(k=None), E_NULL), (dict(cos=None), E_NULL),
    (dict(positions=None), E_NULL), (dict(k_out=None), E_NULL), (dict(q_t=-8), E_SHAPE),
    (dict(q_t=516), E_ALIGN), (dict(k_h=60), E_ALIGN), (dict(q=FAKE + 8), E_ALIGN), (dict(sin=FAKE + 4), E_ALIGN),
    (dict(tokens=0), 0), (dict(tokens=1 << 30, h=60000), E_RANGE)])
def test_rope_refusals(pkg, changes, status):
    assert _call(pkg, "lse_rope", ROPE, changes) == status


@pytest.mark.parametrize("changes,status", [
    (dict(d=96), E_SHAPE), (dict(h=7), E_SHAPE), (dict(h_kv=0), E_SHAPE), (dict(rotary=128), E_SHAPE),
    (dict(rotary=24), E_SHAPE), (dict(block_size=24), E_SHAPE), (dict(block_size=0), E_SHAPE),
    (dict(t_stride=4), E_SHAPE), (dict(stride=2032), E_SHAPE), (dict(s_stride=3), E_SHAPE),
    (dict(entries=-1), E_SHAPE), (dict(most=-1), E_SHAPE), (dict(blocks=-1), E_SHAPE),
    (dict(max_blocks=1 << 30, t_stride=1 << 30), E_RANGE), (dict(k=None), E_NULL), (dict(v_pool=None), E_NULL),
    (dict(scales=None), E_NULL), (dict(q_out=None), E_NULL), (dict(cos=None), E_NULL), (dict(rows=0), E_SHAPE),
    (dict(length=None), E_NULL), (dict(k_t=-64), E_SHAPE), (dict(v_h=60), E_ALIGN), (dict(k=FAKE + 2), E_ALIGN),
    (dict(stride=2056), E_ALIGN), (dict(v_pool=FAKE + 8), E_ALIGN), (dict(entries=0), 0), (dict(tokens=0), 0),
    (dict(most=0), 0)])
def test_append_refusals(pkg, changes, status):
    assert _call(pkg, "lse_append_kv_fp8", APPEND, changes) == status


@pytest.mark.parametrize("changes,status", [
    (dict(d=96), E_SHAPE), (dict(h=7), E_SHAPE), (dict(h=34), E_SHAPE), (dict(block_size=8), E_SHAPE),
    (dict(blocks=0), E_SHAPE), (dict(t_stride=4), E_SHAPE), (dict(stride=2032), E_SHAPE),
    (dict(s_stride=3), E_SHAPE), (dict(q=None), E_NULL), (dict(o=None), E_NULL), (dict(scales=None), E_NULL),
    (dict(ctx=None), E_NULL), (dict(q_h=-256), E_SHAPE), (dict(o_t=60), E_ALIGN), (dict(o=FAKE + 8), E_ALIGN),
    (dict(k_pool=FAKE + 8), E_ALIGN), (dict(stride=2056), E_ALIGN), (dict(s_stride=5), E_ALIGN),
    (dict(scales=FAKE + 1), E_ALIGN), (dict(table=FAKE + 2), E_ALIGN),
    (dict(blocks=1 << 26), E_RANGE),  # a pool of 2^37 bytes a side
    (dict(max_blocks=1 << 28, t_stride=1 << 28), E_RANGE),
    (dict(max_blocks=(1 << 26) + 1, t_stride=1 << 28), E_RANGE),
    (dict(max_blocks=500, t_stride=500), E_WORKSPACE),  # splits, and has no workspace
    (dict(entries=0), 0), (dict(tokens=0), 0), (dict(most=0), 0)])
def test_attention_refusals(pkg, changes, status):
    assert _attend(pkg, changes) == status


def test_workspace_refusals(pkg):
    assert _attend(pkg, {}, None, -1) == E_WORKSPACE
    assert _attend(pkg, {}, FAKE + 8, 1 << 20) == E_WORKSPACE
    split = dict(max_blocks=500, t_stride=500)
    need = _size(pkg, **split)
    assert need > 0
    assert _attend(pkg, split, FAKE, need - 1) == _attend(pkg, split, None, need) == E_WORKSPACE


def _size(pkg, **changes):
    from llm_serving_engine_amd import _lib

    return pkg.library().lse_paged_attention_fp8_workspace_bytes(
        _pack(pkg, _lib.PAGED_ATTENTION_FP8_ARGS, ATTEND, changes))


def test_workspace_sizes(pkg):
    assert _size(pkg, d=96) == _size(pkg, entries=-1) == -1
    assert _size(pkg, entries=0) == 0
    assert _size(pkg, max_blocks=128) == 0  # contexts too short to split
    split = _size(pkg, max_blocks=129)
    assert split == 512 * 16 * (64 + 2) * 4 == _size(pkg, max_blocks=1 << 20)
    assert _size(pkg, entries=4096, tokens=4096, h=32, h_kv=8, d=128, most=1, max_blocks=4096) == 0


def test_tensors_are_checked(pkg):
    """What Python turns down itself: devices, types and shapes of the tensors."""
    ops = pkg.ops
    pool = ops.fp8_kv_pool(4, 16, 2, 64, "cpu")
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="device"):
        ops.append_kv_fp8(None, x, x, None, None, pool, table, i, i, i, 3)
    with pytest.raises(RuntimeError, match="device"):
        ops.paged_attention_fp8(x.transpose(0, 1), pool, table, i, i, i, i, 3)
    with pytest.raises(RuntimeError, match="device"):
        ops.rope(x, None, torch.zeros(4, 32), torch.zeros(4, 32), i)
    bad = [pool._replace(k=pool.k.view(torch.uint8)), pool._replace(scales=pool.scales[:2]),
           pool._replace(v=pool.v[:3]), pool._replace(k=pool.k[..., :512], v=pool.v[..., :512]),
           pool._replace(scales=pool.scales.view(torch.uint8)),
           pool._replace(v=pool.v.flip(0)[::2])]
    wide = ops.fp8_kv_pool(4, 32, 2, 64, "cpu")
    bad += [wide._replace(k=wide.k.transpose(1, 2).contiguous().transpose(1, 2)),
            ops.Fp8KV(wide.k[::2], wide.v[:2], wide.scales[::2])]
    for p in bad:
        with pytest.raises(RuntimeError):
            ops._check_fp8_pool(p)
    assert ops._check_fp8_pool(pool) == (4, 2, 1, 64, 2048, 4)
    assert ops._check_fp8_pool(ops.Fp8KV(*(t[::2] for t in wide))) == (2, 2, 2, 64, 8192, 16)
    assert ops._check_fp8_pool(ops.Fp8KV(*(t[3:] for t in wide))) == (1, 2, 2, 64, 4096, 8)
    for t, e in ((table.long(), i), (table[0], i), (table, torch.zeros(2, dtype=torch.int32)), (table, i.float())):
        with pytest.raises(RuntimeError):
            ops._check_plan(t, e)
    assert ops._check_plan(table, i, i) == (1, 4, 4)
    for cos, sin in ((torch.zeros(4, 32), torch.zeros(4, 31)), (torch.zeros(4, 32).double(), torch.zeros(4, 32)),
                     (torch.zeros(32, 4).t(), torch.zeros(32, 4).t()), (torch.zeros(4, 4),) * 2,
                     (torch.zeros(4, 12),) * 2, (torch.zeros(4, 40),) * 2):
        with pytest.raises(RuntimeError):
            ops._rope_tables(cos, sin, 64)
