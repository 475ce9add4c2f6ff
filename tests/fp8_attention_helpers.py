"""The 8-bit cache's attention through the C entry points: what a call would run, and calls with a caller's own
output, workspace and scale."""

from __future__ import annotations

import ctypes

import torch

FIELDS = ("q", "q_h", "q_t", "k_pool", "v_pool", "stride", "scales", "s_stride", "blocks", "block_size", "table",
          "t_stride", "max_blocks", "ctx", "offset", "start", "length", "o", "o_h", "o_t", "entries", "tokens", "most",
          "h", "h_kv", "d")


def pack(scale=1.0, **fields) -> bytes:
    from llm_serving_engine_amd import _lib

    assert set(fields) <= set(FIELDS)
    return _lib.PAGED_ATTENTION_FP8_ARGS.pack(*(fields.get(n, 0) for n in FIELDS), scale)


def choice(pkg, entries, tokens, most, h, h_kv, d, room, block_size=16) -> tuple[bool, int, int]:
    """(row-tiled, parts, units of split keys) of a call whose table has `room` positions."""
    assert room % block_size == 0
    got = [ctypes.c_int64(-1) for _ in range(3)]
    args = pack(block_size=block_size, max_blocks=room // block_size, entries=entries, tokens=tokens, most=most, h=h,
                h_kv=h_kv, d=d)
    assert pkg.library().lse_paged_attention_fp8_choice(args, *(ctypes.byref(v) for v in got)) == 0
    return bool(got[0].value), got[1].value, got[2].value


def choice_of(pkg, case, most=None) -> tuple[bool, int, int]:
    h, tokens, d = case["q"].shape
    return choice(pkg, len(case["ql"]), tokens, most or int(case["ql"].max()), h, case["pool"][0].shape[1], d,
                  case["table"].shape[1] * case["bs"], case["bs"])


def attend_into(pkg, q, pool, plan, most, o, scale=None, fill=0xff) -> None:
    """One call into the caller's o, with a workspace of `fill` bytes (0xff: NaN in what nobody writes)."""
    table, ctx, qo, qs, ql = plan
    h, tokens, d = q.shape
    per = pool.k.shape[2]
    args = pack(d ** -0.5 if scale is None else scale, q=q.data_ptr(), q_h=q.stride(0), q_t=q.stride(1),
                k_pool=pool.k.data_ptr(), v_pool=pool.v.data_ptr(), stride=pool.k.stride(0),
                scales=pool.scales.data_ptr(), s_stride=pool.scales.stride(0), blocks=pool.k.shape[0],
                block_size=16 * per, table=table.data_ptr(), t_stride=table.stride(0), max_blocks=table.shape[1],
                ctx=ctx.data_ptr(), offset=qo.data_ptr(), start=qs.data_ptr(), length=ql.data_ptr(), o=o.data_ptr(),
                o_h=o.stride(0), o_t=o.stride(1), entries=table.shape[0], tokens=tokens, most=most, h=h,
                h_kv=pool.k.shape[1], d=d)
    lib = pkg.library()
    nbytes = lib.lse_paged_attention_fp8_workspace_bytes(args)
    assert nbytes >= 0
    ws = torch.full((max(nbytes, 16),), fill, dtype=torch.uint8, device=q.device)
    status = lib.lse_paged_attention_fp8(args, ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status == 0
