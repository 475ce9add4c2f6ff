"""The operators of a K/V cache held in 8 bits, as a serving engine calls them, with their plain forms:

  * "rope": rotary positions of a batch's q and k rows from tables of cosines and sines, in the half or the
    interleaved layout, over the whole head or its first `rotary` dims;
  * "append": the same rotation applied to q and k while the batch's k and v rows go into the paged 8-bit
    cache, which keeps a scale for every 16 positions of a head;
  * "attention": causal attention of a batch plan (sequences decoding, prompt chunks, or both) over that
    cache.

The cache (`ops.Fp8KV`): codes k and v, float8 e4m3, (blocks, H_KV, S, 16 D) with S = block_size / 16, and
scales, powers of two (e8m0), (blocks, H_KV, S, 2) for k and v. Position n of a sequence lies in the block
that its table names at n / block_size, group s = n % block_size / 16, slot n % 16. In a group, k[slot][d] is
at ((slot / 4 * D / 64 + d / 64) * 4 + slot % 4) * 64 + d % 64, and v[slot][d] at 16 d + slot.

An appended group's scale is the smallest power of two with every finite value of its slots within 448
scales, at least 2^-126, and at least the group's former scale if it held earlier positions of the sequence,
which are then rounded to the new scale; what is not finite is held as NaN. Slots behind the last appended
position of its group are zeroed.

Heads are those of Llama-3-8B (32 query over 8 K/V heads of 128) and Llama-3.2-3B (24 over 8), with heads of
64 and other groups beside them; an engine iteration holds at most 64 sequences, prompts are cut into chunks
of at most 2048 tokens, blocks have 16 slots unless the engine sets more.
"""

from __future__ import annotations

import math
import random

import torch

own = False

GROUP = 16  # positions that share a scale
F8 = torch.float8_e4m3fn
E8 = torch.float8_e8m0fnu
THETA = 500000.0


def listed():
    llama = dict(h=32, h_kv=8, d=128, rotary=128, interleaved=False, block=16)
    small = dict(h=24, h_kv=8, d=128, rotary=128, interleaved=False, block=16)
    return [
        # One sequence decoding: the smallest call.
        dict(name="rope 1", kind="rope", **llama, decodes=1, chunks=0, chunk=0, ctx=700, lens=1),
        # Three packed prompts in the interleaved layout, half of each head rotated.
        dict(name="rope 3 prompts", kind="rope", **{**llama, "rotary": 64, "interleaved": True},
             decodes=0, chunks=3, chunk=2048, ctx=0, lens=2),
        # A full decode batch: one token of each sequence, mostly into half-filled groups.
        dict(name="append decode 64", kind="append", **llama, decodes=64, chunks=0, chunk=0, ctx=2048,
             lens=3),
        # Fresh prompts of an iteration.
        dict(name="append 3 prompts", kind="append", **llama, decodes=0, chunks=3, chunk=2048, ctx=0,
             lens=4),
        # Continuous batching with heads of 64, blocks of 64 and partial interleaved rotation.
        dict(name="append mixed d64", kind="append",
             **{**llama, "d": 64, "rotary": 32, "interleaved": True, "block": 64}, decodes=40, chunks=1,
             chunk=1024, ctx=2048, lens=5),
        # One sequence decoding behind a short context: the least attention work, all latency.
        dict(name="attention 1", kind="attention", **llama, decodes=1, chunks=0, chunk=0, ctx=500, lens=6),
        # A full decode batch over contexts of different lengths.
        dict(name="attention decode 64", kind="attention", **llama, decodes=64, chunks=0, chunk=0,
             ctx=2048, lens=7),
        # A few long conversations.
        dict(name="attention decode 4 far", kind="attention", **small, decodes=4, chunks=0, chunk=0,
             ctx=60000, lens=8),
        # A full decode batch behind long contexts, heads of 64 in blocks of 32: the most bytes.
        dict(name="attention decode 64 far d64", kind="attention",
             **{**llama, "d": 64, "rotary": 64, "block": 32}, decodes=64, chunks=0, chunk=0, ctx=16384,
             lens=9),
        # Fresh prompts.
        dict(name="attention 3 prompts", kind="attention", **llama, decodes=0, chunks=3, chunk=2048,
             ctx=0, lens=2),
        # A prompt's last chunk behind a long context: the most operations.
        dict(name="attention chunk far", kind="attention", **llama, decodes=0, chunks=1, chunk=2048,
             ctx=12000, lens=10),
        # Continuous batching: a chunk of one prompt beside decoding sequences.
        dict(name="attention mixed", kind="attention", **small, decodes=40, chunks=1, chunk=1024, ctx=2048,
             lens=11),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "attention", "attention", "attention"])
    h, h_kv = rng.choice([(32, 8), (24, 8), (32, 8), (8, 8), (16, 1), (10, 2)])
    d = rng.choice([128, 128, 64])
    rotary = rng.choice([d, d, d // 2, d // 4])
    case = dict(kind=kind, h=h, h_kv=h_kv, d=d, rotary=rotary, interleaved=rng.random() < 0.4,
                block=rng.choice([16, 16, 32, 64, 48]), lens=rng.randrange(1 << 20))
    what = rng.choice(["decode", "prompts", "mixed"])
    if what == "decode":
        decodes = _log(rng, 1, 64)
        return dict(case, decodes=decodes, chunks=0, chunk=0, ctx=_log(rng, 20, 200000 // max(decodes, 4)))
    chunk = _log(rng, 2, 2048)
    chunks = rng.randint(1, max(1, min(4, 4096 // chunk)))
    ctx = rng.choice([0, _log(rng, 64, 2048)])
    if what == "prompts":
        return dict(case, decodes=0, chunks=chunks, chunk=chunk, ctx=ctx)
    return dict(case, decodes=_log(rng, 1, 60), chunks=1, chunk=chunk, ctx=max(ctx, 64))


# ---- inputs ------------------------------------------------------------------------------------


def _entries(case) -> list[tuple[int, int]]:
    """(new tokens, positions before them) of every sequence of the call, prompt chunks first."""
    r = random.Random(case["lens"])
    got = []
    for _ in range(case["chunks"]):
        rows = r.randint(max(1, (3 * case["chunk"]) // 5), case["chunk"])
        got.append((rows, r.randint(case["ctx"] // 2, case["ctx"]) if case["ctx"] else 0))
    for _ in range(case["decodes"]):
        got.append((1, r.randint(max(1, case["ctx"] // 8), case["ctx"]) - 1))
    return got


def _gen(seed: int, what: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(16 * seed + what)


def _tables(case, n: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Cosines and sines (n, rotary / 2) of positions 0 .. n - 1, as a model keeps them."""
    half = torch.arange(0, case["rotary"], 2, device="cuda", dtype=torch.float64) / case["rotary"]
    angle = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] / THETA ** half
    return torch.cos(angle).float(), torch.sin(angle).float()


def _codes(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Groups x (..., 16, d) as codes of the same shape and e8m0 bytes (...)."""
    bits = x.abs().amax((-1, -2)).view(torch.int32)
    e = torch.clamp(((bits + 0x1FFFFF) >> 23) - 8, min=1)
    return (x * torch.exp2((127 - e).float())[..., None, None]).to(F8), e.to(torch.uint8)


def _pack_k(c: torch.Tensor) -> torch.Tensor:
    """Codes (..., 16, d) in the order that k has them in."""
    lead, d = c.shape[:-2], c.shape[-1]
    return c.reshape(*lead, 4, 4, d // 64, 64).transpose(-3, -2).reshape(*lead, 16 * d)


def _unpack_k(c: torch.Tensor, d: int) -> torch.Tensor:
    lead = c.shape[:-1]
    return c.reshape(*lead, 4, d // 64, 4, 64).transpose(-3, -2).reshape(*lead, 16, d)


def _pack_v(c: torch.Tensor) -> torch.Tensor:
    return c.transpose(-1, -2).reshape(*c.shape[:-2], -1)


def _unpack_v(c: torch.Tensor, d: int) -> torch.Tensor:
    return c.reshape(*c.shape[:-1], d, 16).transpose(-1, -2)


def prepare(case, seed):
    entries, d, h_kv = _entries(case), case["d"], case["h_kv"]
    rows = [n for n, _ in entries]
    tokens = sum(rows)
    before = [c for _, c in entries]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    start = [sum(rows[:e]) for e in range(len(rows))]
    cos, sin = _tables(case, max(n + c for n, c in entries))
    g = _gen(seed, 0)
    # The stacked projection's output; a few channels of k are several times larger, as trained models have.
    qkv = torch.randn(tokens, case["h"] + 2 * h_kv, d, generator=g, device="cuda")
    loud = 1.0 + 7.0 * (torch.rand(h_kv, d, generator=g, device="cuda") < 0.03)
    qkv[:, case["h"]:case["h"] + h_kv] *= loud
    qkv = qkv.to(torch.bfloat16)
    state = dict(case=case, q=qkv[:, :case["h"]], k=qkv[:, case["h"]:case["h"] + h_kv],
                 v=qkv[:, case["h"] + h_kv:], cos=cos, sin=sin)
    if case["kind"] == "rope":
        state["positions"] = i32([c + m for n, c in entries for m in range(n)])
        return state
    per = case["block"] // GROUP
    need = [-(-(n + c) // case["block"]) for n, c in entries]
    blocks = sum(need) + 1
    perm = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros(len(entries), max(need), dtype=torch.int32)
    at = 0
    for e, n in enumerate(need):
        table[e, :n] = perm[at:at + n]
        at += n
    codes = []
    for what in range(2):
        x = torch.randn(blocks, h_kv, per, GROUP, d, generator=_gen(seed, 1 + what), device="cuda")
        if what == 0:
            x *= loud[:, None, None]
        codes.append(_codes(x))
        del x
    state |= dict(pool_k=_pack_k(codes[0][0].view(torch.uint8)).view(F8),
                  pool_v=_pack_v(codes[1][0].view(torch.uint8)).view(F8),
                  scales=torch.stack([codes[0][1], codes[1][1]], -1).view(E8), table=table.cuda(),
                  context_len=i32([n + c for n, c in entries]), query_offset=i32(before),
                  q_start=i32(start), q_len=i32(rows), most=max(rows), seed=seed)
    return state


# ---- the plain forms ---------------------------------------------------------------------------


def _rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x (tokens, heads, d) in 32 bits, cos and sin (tokens, rotary / 2)."""
    half = cos.shape[-1]
    x = x.float()
    c, s = cos[:, None], sin[:, None]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        got = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        got = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([got, rest], -1)


def _byte_scale(e: torch.Tensor) -> torch.Tensor:
    return torch.exp2(e.float() - 127.0)


def _plain_rope(s):
    at = s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    inter = s["case"]["interleaved"]
    return tuple(_rotate(s[n], cos, sin, inter).to(torch.bfloat16) for n in ("q", "k"))


def _k_at(pool, block, sub, slot, d: int):
    """k (blocks, h_kv, groups of a block, 16 d) as a view, and the index of rows (..., h_kv, d / 64, 64)."""
    return pool.unflatten(-1, (4, d // 64, 4, 64)), (block, slice(None), sub, slot // 4, slice(None), slot % 4)


def _v_at(pool, block, sub, slot, d: int):
    """v as a view, and the index of rows (..., h_kv, d)."""
    return pool.unflatten(-1, (d, GROUP)), (block, slice(None), sub, slice(None), slot)


def _plain_append_half(pool, scales, x, new, first, tail, at):
    """x (tokens, h_kv, d) into codes `pool` and their e8m0 bytes `scales` (blocks, h_kv, groups of a block).
    new: (block, group, slot) of every token; first, tail: those of all 16 slots of each sequence's first and
    last group, with whether a slot is kept, or zeroed."""
    d = x.shape[-1]
    per, (block, sub, slot) = scales.shape[2], new
    old = scales.transpose(1, 2).flatten(0, 1).int()  # (groups, h_kv)
    amax = torch.zeros(old.shape, device=x.device)
    group = block * per + sub
    amax = amax.scatter_reduce(0, group[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    need = torch.clamp(((amax.view(torch.int32) + 0x1FFFFF) >> 23) - 8, min=1)
    touched = torch.zeros(len(old), dtype=torch.bool, device=x.device)
    touched[group] = True
    *where, keep = first
    head = where[0][:, 0] * per + where[1][:, 0]
    kept = torch.zeros_like(touched)
    kept[head] = keep.any(1)
    need = torch.where(kept[:, None], torch.maximum(need, old), need)
    new_scale = torch.where(touched[:, None], need, old)
    # The kept slots of half-filled groups, from the former scale to the new one.
    view, index = at(pool, *where, d)
    rows = view[index]  # (sequences, 16, h_kv, ...)
    ratio = _byte_scale(127 + old[head] - new_scale[head])
    ratio = ratio.reshape(len(head), 1, -1, *[1] * (rows.dim() - 3))
    keep = keep.reshape(*keep.shape, *[1] * (rows.dim() - 2))
    view[index] = torch.where(keep, (rows.view(F8).float() * ratio).to(F8).view(torch.uint8), rows)
    view, index = at(pool, *new, d)
    codes = (x * _byte_scale(254 - new_scale[group])[..., None]).to(F8).view(torch.uint8)
    view[index] = codes.reshape(view[index].shape)
    *where, clear = tail
    view, index = at(pool, *where, d)
    rows = view[index]
    clear = clear.reshape(*clear.shape, *[1] * (rows.dim() - 2))
    view[index] = torch.where(clear, torch.zeros_like(rows), rows)
    scales.copy_(new_scale.to(torch.uint8).unflatten(0, (-1, per)).transpose(1, 2))


def _plain_append(s):
    c = s["case"]
    tokens, block = s["q"].shape[0], c["block"]
    n, offset = s["q_len"].long(), s["query_offset"].long()
    every = torch.arange(len(n), device="cuda")
    entry = torch.repeat_interleave(every, n, output_size=tokens)
    pos = offset[entry] + torch.arange(tokens, device="cuda") - s["q_start"].long()[entry]
    place = lambda e, p: (s["table"].long()[e, p // block], p % block // GROUP, p % GROUP)  # noqa: E731
    slots = torch.arange(GROUP, device="cuda")[None]
    head = (offset // GROUP * GROUP)[:, None] + slots
    last = ((offset + n - 1) // GROUP * GROUP)[:, None] + slots
    first = (*place(every[:, None], head), head < offset[:, None])
    tail = (*place(every[:, None], last), last >= (offset + n)[:, None])
    q, k = (_rotate(s[x], s["cos"][pos], s["sin"][pos], c["interleaved"]) for x in ("q", "k"))
    scales = s["scales"].view(torch.uint8)
    for what, (x, pool, at) in enumerate([(k, "pool_k", _k_at), (s["v"].float(), "pool_v", _v_at)]):
        _plain_append_half(s[pool].view(torch.uint8), scales[..., what], x, place(entry, pos), first, tail, at)
    return q.to(torch.bfloat16), s["pool_k"], s["pool_v"], s["scales"]


def _cached(s, table, width: int, pool: str, what: int, unpack):
    """A sequence batch's K or V (entries, h_kv, width, d) in 32 bits."""
    c = s["case"]
    codes = s[pool].view(torch.uint8)[table]  # (entries, blocks, h_kv, groups, 16 d)
    x = unpack(codes, c["d"]).contiguous().view(F8).float()
    x = x * _byte_scale(s["scales"].view(torch.uint8)[..., what][table])[..., None, None]
    x = x.permute(0, 2, 1, 3, 4, 5).reshape(len(table), c["h_kv"], -1, c["d"])
    return x[:, :, :width]


def _plain_attend(s, lo: int, hi: int, rows: list[int], width: int):
    """Entries lo .. hi of `rows` rows each behind contexts of at most `width`: (h, their rows, d)."""
    c = s["case"]
    most, g = max(rows), c["h"] // c["h_kv"]
    table = s["table"][lo:hi, :-(-width // c["block"])].long()
    k = _cached(s, table, width, "pool_k", 0, _unpack_k)
    v = _cached(s, table, width, "pool_v", 1, _unpack_v)
    m = torch.arange(most, device="cuda")
    start, n, ctx, offset = (s[x][lo:hi].long()[:, None] for x in
                             ("q_start", "q_len", "context_len", "query_offset"))
    real = m[None] < n
    q = s["q"][torch.where(real, start + m, start)].float()  # (entries, most, h, d)
    q = q.reshape(hi - lo, most, c["h_kv"], g, c["d"]).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(hi - lo, c["h_kv"], g * most, c["d"]), k.transpose(-1, -2).contiguous())
    score = score.view(hi - lo, c["h_kv"], g, most, width) * (1.0 / math.sqrt(c["d"]))
    at = torch.arange(width, device="cuda")
    seen = (at[None, None] <= (offset + m)[..., None]) & (at[None, None] < ctx[..., None])
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    v = torch.where((at[None] < ctx)[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.view(hi - lo, c["h_kv"], g * most, width), v).view(*total.shape[:-1], c["d"]) / total
    o = o.permute(1, 2, 0, 3, 4).reshape(c["h"], (hi - lo) * most, c["d"])
    index = torch.cat([e * most + torch.arange(r, device="cuda") for e, r in enumerate(rows)])
    return o[:, index].to(torch.bfloat16)


def _plain_attention(s):
    """Prompt chunks and decoding sequences each as one padded batch."""
    c, entries = s["case"], _entries(s["case"])
    got = []
    for lo, hi in ((0, c["chunks"]), (c["chunks"], len(entries))):
        if hi > lo:
            part = entries[lo:hi]
            got.append(_plain_attend(s, lo, hi, [n for n, _ in part], max(n + b for n, b in part)))
    return torch.cat(got, 1) if len(got) > 1 else got[0]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention}[c["kind"]](s)
    import __graft_entry__

    ops = __graft_entry__.load_package().ops
    if c["kind"] == "rope":
        return ops.rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], interleaved=c["interleaved"])
    pool = ops.Fp8KV(s["pool_k"], s["pool_v"], s["scales"])
    if c["kind"] == "append":
        q = ops.append_kv_fp8(s["q"], s["k"], s["v"], s["cos"], s["sin"], pool, s["table"],
                              s["query_offset"], s["q_start"], s["q_len"], s["most"],
                              interleaved=c["interleaved"])
        return q, pool.k, pool.v, pool.scales
    # The output comes in q's own token-major layout; (h, tokens, d) is a view of it.
    return ops.paged_attention_fp8(s["q"].transpose(0, 1), pool, s["table"], s["context_len"],
                                   s["query_offset"], s["q_start"], s["q_len"], s["most"])


# ---- what a pass cannot do without -------------------------------------------------------------


def work(case):
    entries = _entries(case)
    tokens, d, h, h_kv = sum(n for n, _ in entries), case["d"], case["h"], case["h_kv"]
    tables = 4 * case["rotary"] * tokens  # a row of cosines and one of sines per token
    if case["kind"] == "rope":
        return dict(bytes=4 * tokens * (h + h_kv) * d + tables + 4 * tokens,
                    flops=3 * tokens * (h + h_kv) * case["rotary"])
    if case["kind"] == "append":
        # q in and out, k and v in, their codes out; the scales, and of half-filled groups the old ones in.
        groups = sum((c + n - 1) // GROUP - c // GROUP + 1 for n, c in entries)
        halves = sum(c % GROUP > 0 for _, c in entries)
        return dict(bytes=4 * tokens * h * d + 6 * tokens * h_kv * d + tables + 2 * (groups + halves) * h_kv,
                    flops=3 * tokens * (h + h_kv) * case["rotary"] + 4 * tokens * h_kv * d)
    cached = sum(n + c for n, c in entries)
    scales = sum(-(-(n + c) // GROUP) for n, c in entries)
    seen = sum(n * c + n * (n + 1) // 2 for n, c in entries)  # row r sees the positions up to its own
    return dict(bytes=2 * cached * h_kv * d + 2 * scales * h_kv + 4 * tokens * h * d,
                flops=4 * d * h * seen)


# ---- the same in 64 bits -----------------------------------------------------------------------


def _e4m3(x: torch.Tensor) -> torch.Tensor:
    """x (64 bits, within 448) to the nearest e4m3 value, ties to even: steps of 2^(e - 3), e at least -6."""
    _, e = torch.frexp(x)
    step = torch.exp2(torch.clamp(e - 1, min=-6).double() - 3)
    return torch.round(x / step) * step


def _exact_turn(x: torch.Tensor, case, at: torch.Tensor, cos, sin) -> torch.Tensor:
    """x (tokens, heads, d), token t rotated to position at[t]: pair by pair, as complex products."""
    x = x.double()
    turn = torch.complex(cos[at].double(), sin[at].double())[:, None]
    r = case["rotary"]
    i = torch.arange(r // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
    z = torch.complex(x[..., a], x[..., b]) * turn
    out = x.clone()
    out[..., a], out[..., b] = z.real, z.imag
    return out


def _exact_values(s, e: int, n: int, what: int) -> torch.Tensor:
    """Positions 0 .. n - 1 of entry e: (n, h_kv, d)."""
    c = s["case"]
    p = torch.arange(n, device="cuda")
    block, group = s["table"][e].long()[p // c["block"]], p % c["block"] // GROUP
    slot, dd = (p % GROUP)[:, None], torch.arange(c["d"], device="cuda")[None]
    if what == 0:
        inner = ((slot // 4 * (c["d"] // 64) + dd // 64) * 4 + slot % 4) * 64 + dd % 64
    else:
        inner = 16 * dd + slot
    codes = s[("pool_k", "pool_v")[what]].view(torch.uint8)
    got = torch.empty(n, c["h_kv"], c["d"], dtype=torch.float64, device="cuda")
    for head in range(c["h_kv"]):
        rows = codes[block, head, group]
        scale = s["scales"].view(torch.uint8)[block, head, group, what].double() - 127
        got[:, head] = rows.gather(1, inner).view(F8).double() * torch.exp2(scale)[:, None]
    return got


def _exact_append(s):
    c = s["case"]
    k_new, q_new = [], []
    for e, (n, before) in enumerate(_entries(c)):
        a = int(s["q_start"][e])
        at = torch.arange(before, before + n, device="cuda")
        q_new.append(_exact_turn(s["q"][a:a + n], c, at, s["cos"], s["sin"]))
        k_new.append(_exact_turn(s["k"][a:a + n], c, at, s["cos"], s["sin"]))
    pools = []
    scales = torch.exp2(s["scales"].view(torch.uint8).double() - 127)
    for what, name in enumerate(("pool_k", "pool_v")):
        pool = s[name].double()
        for e, (n, before) in enumerate(_entries(c)):
            a = int(s["q_start"][e])
            new = k_new[e] if what == 0 else s["v"][a:a + n].double()
            for g in range(before // GROUP, (before + n - 1) // GROUP + 1):
                block = int(s["table"][e, g * GROUP // c["block"]])
                inner = g % (c["block"] // GROUP)
                x = torch.zeros(c["h_kv"], GROUP, c["d"], dtype=torch.float64, device="cuda")
                lo, hi = max(before - g * GROUP, 0), min(before + n - g * GROUP, GROUP)
                x[:, lo:hi] = new[g * GROUP + lo - before:g * GROUP + hi - before].transpose(0, 1)
                top = x.abs().amax((1, 2))
                scale = torch.exp2(torch.ceil(torch.log2(top / 448)))
                scale = torch.clamp(torch.where(top / 448 > scale, 2 * scale, scale), min=2.0 ** -126)
                if lo:
                    unpack = _unpack_k if what == 0 else _unpack_v
                    former = unpack(pool[block, :, inner], c["d"])[:, :lo]
                    was = scales[block, :, inner, what]
                    scale = torch.maximum(scale, was)
                    x[:, :lo] = former * was[:, None, None]
                codes = _e4m3(x / scale[:, None, None])
                pool[block, :, inner] = (_pack_k if what == 0 else _pack_v)(codes)
                scales[block, :, inner, what] = scale
        pools.append(pool)
    return torch.cat(q_new), *pools, scales


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        at = s["positions"].long()
        return tuple(_exact_turn(s[n], case, at, s["cos"], s["sin"]) for n in ("q", "k"))
    if case["kind"] == "append":
        return _exact_append(s)
    out = torch.empty(case["h"], s["q"].shape[0], case["d"], dtype=torch.float64, device="cuda")
    g = case["h"] // case["h_kv"]
    for e, (n, before) in enumerate(_entries(case)):
        a = int(s["q_start"][e])
        k, v = (_exact_values(s, e, n + before, what).transpose(0, 1).contiguous() for what in (0, 1))
        hide = torch.arange(n + before, device="cuda")[None] > before + torch.arange(n, device="cuda")[:, None]
        for head in range(case["h"]):
            score = s["q"][a:a + n, head].double() @ k[head // g].t().contiguous() / math.sqrt(case["d"])
            p = torch.softmax(score.masked_fill(hide, -math.inf), -1)
            out[head, a:a + n] = p @ v[head // g]
    return out
