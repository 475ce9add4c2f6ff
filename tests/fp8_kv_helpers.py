"""Cases for the 8-bit K/V cache's tests: plans, pools and their fp64 results."""

from __future__ import annotations

import numpy as np
import torch

from helpers import bf16_bits, to_bf16_tensor
from oracle import kv_cache as kv
from oracle import numerics as ora


def bf16_rows(rng, *shape, scale=1.0):
    """fp32 values that are bf16 ones."""
    return ora.bf16_bits_to_f32(ora.f32_to_bf16_bits((rng.standard_normal(shape) * scale).astype(np.float32)))


def to_dev(x: np.ndarray, dev):
    return to_bf16_tensor(ora.f32_to_bf16_bits(x.astype(np.float32)), dev)


def i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)


def plan_of(rng, entries, block_size, spare=2):
    """entries: (q_len, query_offset, context_len). Blocks shuffled over one pool with `spare` of nobody."""
    ql, qo, ctx = (np.array([e[i] for e in entries], np.int32) for i in range(3))
    need = [max(1, -(-max(int(c), int(o) + int(n)) // block_size)) for n, o, c in entries]
    perm = rng.permutation(sum(need) + spare)
    table = np.zeros((len(entries), max(need)), np.int32)
    at = 0
    for e, n in enumerate(need):
        table[e, :n] = perm[at:at + n]
        at += n
    qs = np.concatenate([[0], np.cumsum(ql)[:-1]]).astype(np.int32)
    return dict(table=table, qo=qo, ctx=ctx, qs=qs, ql=ql, blocks=len(perm))


def random_pool(rng, blocks, block_size, n_kv, d, loud=1.0):
    """(k codes, v codes, scales) of groups of normal values, scales as the append chooses them."""
    per = block_size // kv.GROUP
    codes, scales = [], np.empty((blocks, n_kv, per, 2), np.uint8)
    slot, dim = np.meshgrid(np.arange(kv.GROUP), np.arange(d), indexing="ij")
    for what, index in enumerate((kv.k_index, kv.v_index)):
        x = rng.standard_normal((blocks, n_kv, per, kv.GROUP, d)) * (loud if what == 0 else 1.0)
        x *= 2.0 ** rng.integers(-3, 4, (blocks, n_kv, per, 1, 1))  # scales that differ
        scales[..., what] = kv.scale_byte(np.abs(x).max((-1, -2)))
        x = x * 2.0 ** (127.0 - scales[..., what])[..., None, None]
        out = np.empty((blocks, n_kv, per, kv.GROUP * d), np.uint8)
        out[..., index(slot, dim, d)] = kv.encode(x)
        codes.append(out)
    return codes[0], codes[1], scales


def pool_to_dev(pkg, pool, dev):
    k, v, s = (torch.from_numpy(a.copy()).to(dev) for a in pool)
    return pkg.ops.Fp8KV(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn),
                         s.view(torch.float8_e8m0fnu))


def pool_to_host(pool):
    return tuple(t.view(torch.uint8).cpu().numpy() for t in pool)


def same_pool(got, want):
    """Equal bytes, any NaN code as good as another."""
    for name, a, b in zip(("k", "v"), got[:2], want[:2]):
        nan = (a & 127 == 127) & (b & 127 == 127)
        differ = (a != b) & ~nan
        assert not differ.any(), f"{name}: {int(differ.sum())} codes differ, first at {np.argwhere(differ)[0]}"
    np.testing.assert_array_equal(got[2], want[2])


def attend_args(case, dev):
    return [i32(case[n], dev) for n in ("table", "ctx", "qo", "qs", "ql")]


def attend(pkg, dev, case, most=None):
    o = pkg.ops.paged_attention_fp8(to_bf16_tensor(case["q"], dev), pool_to_dev(pkg, case["pool"], dev),
                                    *attend_args(case, dev), most or int(case["ql"].max()))
    torch.cuda.synchronize()
    return bf16_bits(o)


def attention_case(seed, entries, h=32, h_kv=8, d=128, block_size=16, q_scale=1.0):
    rng = np.random.default_rng(seed)
    case = plan_of(rng, entries, block_size)
    tokens = int(case["ql"].sum())
    case["q"] = ora.f32_to_bf16_bits((rng.standard_normal((h, tokens, d)) * q_scale).astype(np.float32))
    case["pool"] = random_pool(rng, case["blocks"], block_size, h_kv, d)
    case["bs"] = block_size
    return case


def attention_golden(case):
    """(fp64 result, covered rows, largest |V|): what a pool stands for is exact in bf16. Rows of entries
    without a context are not covered."""
    k, v = (x.astype(np.float32) for x in kv.unpack(case["pool"], case["bs"]))
    bits = [ora.f32_to_bf16_bits(x) for x in (k, v)]
    for x, b in zip((k, v), bits):
        np.testing.assert_array_equal(ora.bf16_bits_to_f32(b), x)
    golden, covered = ora.paged_attention_golden(case["q"], *bits, case["table"], case["ctx"], case["qo"],
                                                 case["qs"], np.where(case["ctx"] > 0, case["ql"], 0),
                                                 case["bs"])
    return golden, covered, float(np.nanmax(np.abs(v)))


def check_attention(pkg, dev, case, what="", most=None):
    """|o - golden| <= 2^-8 (max|V| + |golden|): a probability is rounded to bf16 (2^-9 of it, the output
    being a convex combination of V rows) and so is the output."""
    o = attend(pkg, dev, case, most)
    golden, covered, vmax = attention_golden(case)
    ok, msg = ora.attention_within_tolerance(o, golden, vmax, covered)
    assert ok, f"{what}: {msg}"
    return o
