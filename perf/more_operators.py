"""The operators of decoder layers with 4-bit weights, as a serving engine calls them, with their plain forms:

  * "linear": y = x W^T for bf16 rows x and a 4-bit weight W (a projection);
  * "glu": h = silu(x G^T) * (x U^T) for two stacked 4-bit weights (an MLP's gate and up projections);
  * "rows linear": the first with x rounded to 8 bits before it (what o_proj and down_proj call);
  * "rows glu": the second over rows that are held in 8 bits already;
  * "norm": the residual's addition and the root-mean-square norm after it, whose output is held in 8 bits
    (what the rows of q/k/v, gate and up come from).

A 4-bit weight (N, K) holds float4 e2m1 codes, sign and the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6, and for every
32 consecutive k of a row a power of two (e8m0), the smallest from 2^-126 up with the group within 6 scales.
`ops.Fp4Weight` keeps it in tiles: code byte 16 l + i of tile (n / 16, k / 128) holds rows n = 16 .. + l % 16 at
k = 128 .. + 32 (l / 16) + 2 i (low half) and the k after it; scale byte 4 l + t of tile (n / 16, k / 512) belongs
to row l % 16 and the 32 k from 512 .. + 128 t + 32 (l / 16) on. Two stacked weights (2 I, K) take turns by row
tiles of 16: gate, up, gate, up.

Rows in 8 bits (`ops.Fp8Rows`) are float8 e4m3 codes (M, K) and a power of two for every 32 k (M, K / 32), by the
same rule with 448 in place of 6. The norm rounds where a bf16 model does: the sum, the normed value and its product
with the weight go to bf16 each.

Sizes are those of Llama-3-8B (hidden 4096, 14336 in the MLP, 6144 rows of q, k and v) and their shards over 2 to 8
GPUs; an engine iteration decodes at most 64 sequences and takes prompts in chunks of at most 2048 tokens.
"""

from __future__ import annotations

import math
import random

import torch

own = False

GROUP = 32  # weights, or values of a row, that share a scale
F8 = torch.float8_e4m3fn
E8 = torch.float8_e8m0fnu
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-5


def listed():
    return [
        # One sequence decoding, its o_proj: the smallest product, all latency.
        dict(name="linear 1", kind="linear", m=1, n=4096, k=4096),
        # Some sequences decoding: the stacked q/k/v.
        dict(name="linear 13", kind="linear", m=13, n=6144, k=4096),
        # A full decode batch's down_proj.
        dict(name="linear 64 deep", kind="linear", m=64, n=4096, k=14336),
        # A prompt chunk over a weight whose sides are no multiples of a tile.
        dict(name="linear 777", kind="linear", m=777, n=2330, k=4128),
        # A few sequences decoding: the MLP's first half.
        dict(name="glu 5", kind="glu", m=5, n=14336, k=4096),
        # A whole prompt chunk: the most operations.
        dict(name="glu 2048", kind="glu", m=2048, n=14336, k=4096),
        # A full decode batch's o_proj over rows in 8 bits.
        dict(name="rows linear 64", kind="rows linear", m=64, n=4096, k=4096),
        # A whole prompt chunk's down_proj.
        dict(name="rows linear 2048", kind="rows linear", m=2048, n=4096, k=14336),
        # A decode batch's MLP, and a whole prompt chunk's.
        dict(name="rows glu 24", kind="rows glu", m=24, n=14336, k=4096),
        dict(name="rows glu 2048", kind="rows glu", m=2048, n=14336, k=4096),
        # A decode batch's norm, nearly all latency, and that of the longest iteration.
        dict(name="norm 33", kind="norm", m=33, n=0, k=4096),
        dict(name="norm 4160", kind="norm", m=4160, n=0, k=4096),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "glu", "rows linear", "rows glu", "norm"])
    m = _log(rng, 1, rng.choice([64, 2048]))
    if kind == "norm":
        return dict(kind=kind, m=_log(rng, 1, 4160), n=0, k=32 * _log(rng, 16, 448))
    k = rng.choice([4096, 14336, 2048, 7168, 1792, 512, 32 * rng.randint(9, 300)])
    n = rng.choice([4096, 6144, 1024, 768, 512, _log(rng, 100, 6000)])
    if "glu" in kind:
        n, k = rng.choice([14336, 7168, 3584, 1792, _log(rng, 100, 8000)]), min(k, 4096)
    return dict(kind=kind, m=m, n=n, k=k)


# ---- inputs ------------------------------------------------------------------------------------


def _gen(seed: int, what: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(16 * seed + what)


def _scale_bytes(amax: torch.Tensor, most: float) -> torch.Tensor:
    """e8m0 bytes of the smallest powers of two from 2^-126 up that hold amax within `most` of them. most is
    1.75 (448) or 1.5 (6) times a power of two, so the mantissa's bits say which of two neighbours it is."""
    bits = amax.view(torch.int32)
    mantissa, exponent = math.frexp(most)  # most = (2 mantissa) 2^(exponent - 1)
    limit = int((2 * mantissa - 1) * (1 << 23))
    e = (bits >> 23) + ((bits & 0x7FFFFF) > limit) - (exponent - 1)
    return torch.clamp(e, min=1)


def _power(e: torch.Tensor) -> torch.Tensor:
    return torch.exp2(e.float() - 127.0)


def _to_fp4(x: torch.Tensor) -> torch.Tensor:
    """x within 6 to the nearest e2m1 codes, ties to even codes."""
    a = x.abs()
    code = torch.zeros_like(x, dtype=torch.uint8)
    for i in range(1, 8):
        middle = (FP4[i - 1] + FP4[i]) / 2
        code += (a > middle) if i % 2 else (a >= middle)
    return code | ((x < 0) & (code > 0)).to(torch.uint8) << 3


def _pack(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """w (rows, K) in 32 bits as 4-bit tiles: codes (rows / 16, K / 128, 1024), scales (rows / 16, K / 512, 256)."""
    rows, k = w.shape
    groups = w.view(rows, k // GROUP, GROUP)
    e = _scale_bytes(groups.abs().amax(-1), 6.0)
    code = _to_fp4(groups / _power(e)[..., None]).view(rows, k)
    code = torch.nn.functional.pad(code, (0, -k % 128, 0, -rows % 16))
    code = code.view(-1, 16, code.shape[1] // 128, 4, 32).permute(0, 2, 3, 1, 4)
    code = (code[..., 0::2] | code[..., 1::2] << 4).reshape(code.shape[0], code.shape[1], 1024)
    e = torch.nn.functional.pad(e, (0, -(k // GROUP) % 16, 0, -rows % 16), value=127).to(torch.uint8)
    e = e.view(-1, 16, e.shape[1] // 16, 4, 4).permute(0, 2, 4, 1, 3)
    return code, e.reshape(e.shape[0], e.shape[1], 256)


def _take_turns(w: torch.Tensor) -> torch.Tensor:
    """Stacked (2 I, K) as row tiles gate, up, gate, up, each half filled up to whole tiles with zeros."""
    i, k = w.shape[0] // 2, w.shape[1]
    halves = torch.nn.functional.pad(w.view(2, i, k), (0, 0, 0, -i % 16))
    return halves.view(2, -1, 16, k).transpose(0, 1).reshape(-1, k)


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (rows, K) as e4m3 codes and e8m0 bytes (rows, K / 32)."""
    groups = x.float().view(x.shape[0], -1, GROUP)
    e = _scale_bytes(groups.abs().amax(-1), 448.0)
    return (groups / _power(e)[..., None]).to(F8).view(x.shape), e.to(torch.uint8)


def prepare(case, seed):
    m, n, k, kind = case["m"], case["n"], case["k"], case["kind"]
    g = _gen(seed, 0)
    # Activations: a few channels are many times larger than the others, as in trained models.
    loud = 1.0 + 20.0 * (torch.rand(k, generator=g, device="cuda") < 0.005)
    x = (torch.randn(m, k, generator=g, device="cuda") * loud).to(torch.bfloat16)
    state = dict(case=case, x=x)
    if kind == "norm":
        state["residual"] = (4 * torch.randn(m, k, generator=g, device="cuda") * loud).to(torch.bfloat16)
        state["weight"] = (0.5 + torch.rand(k, generator=g, device="cuda")).to(torch.bfloat16)
        return state
    if kind == "rows glu":
        codes, e = _rows(x)
        del state["x"]
        state |= dict(codes8=codes, scales8=e.view(E8))
    stacked = 2 * n if "glu" in kind else n
    # Rows of a trained weight differ in size.
    w = torch.randn(stacked, k, generator=_gen(seed, 1), device="cuda")
    w *= 0.02 * torch.exp(0.5 * torch.randn(stacked, 1, generator=g, device="cuda"))
    codes, scales = _pack(_take_turns(w) if "glu" in kind else w)
    return state | dict(codes=codes, scales=scales.view(E8))


# ---- the plain forms ---------------------------------------------------------------------------


def _plain_weight(s) -> torch.Tensor:
    """The 4-bit weight's packed rows (16 row tiles, K) in 32 bits."""
    codes, scales, k = s["codes"], s["scales"].view(torch.uint8), s["case"]["k"]
    rb, steps = codes.shape[:2]
    value = torch.tensor([*FP4, *(-v for v in FP4)], device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], -1).view(rb, steps, 4, 16, 32)
    w = value[both.permute(0, 3, 1, 2, 4).reshape(rb * 16, steps * 128)[:, :k].int()]
    e = scales.view(rb, -1, 4, 16, 4).permute(0, 3, 1, 4, 2).reshape(rb * 16, -1)[:, :k // GROUP]
    return (w.view(rb * 16, -1, GROUP) * _power(e)[..., None]).view(rb * 16, k)


def _plain_product(s, x: torch.Tensor) -> torch.Tensor:
    """x (M, K) in 32 bits times the weight; for stacked weights with the gate's silu times up."""
    n = s["case"]["n"]
    y = torch.matmul(x, _plain_weight(s).t())
    if "glu" not in s["case"]["kind"]:
        return y[:, :n].to(torch.bfloat16)
    gate, up = y.view(len(y), -1, 2, 16).unbind(2)
    gate, up = gate.reshape(len(y), -1)[:, :n], up.reshape(len(y), -1)[:, :n]
    return (gate / (1 + torch.exp(-gate)) * up).to(torch.bfloat16)


def _plain_rows(codes: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    return (codes.float().view(len(codes), -1, GROUP) * _power(e.view(torch.uint8))[..., None]).view(codes.shape)


def _plain_norm(s):
    hidden = (s["x"].float() + s["residual"].float()).to(torch.bfloat16)
    h = hidden.float()
    normed = (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)).to(torch.bfloat16)
    codes, e = _rows((normed.float() * s["weight"].float()).to(torch.bfloat16))
    return hidden, codes, e.view(E8)


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        if kind == "norm":
            return _plain_norm(s)
        if kind == "rows glu":
            return _plain_product(s, _plain_rows(s["codes8"], s["scales8"]))
        return _plain_product(s, s["x"].float() if kind in ("linear", "glu") else _plain_rows(*_rows(s["x"])))
    import __graft_entry__

    ops = __graft_entry__.load_package().ops
    if kind == "norm":
        hidden, rows = ops.add_rmsnorm_fp8(s["x"], s["residual"], s["weight"], EPS)
        return hidden, rows.codes, rows.scales
    weight = ops.Fp4Weight(s["codes"], s["scales"], s["case"]["n"], s["case"]["k"])
    if kind == "linear":
        return ops.w4a16_linear(s["x"], weight)
    if kind == "glu":
        return ops.w4a16_glu(s["x"], weight)
    if kind == "rows linear":
        return ops.w4a8_linear(ops.quantize_rows_fp8(s["x"]), weight)
    return ops.w4a8_glu(ops.Fp8Rows(s["codes8"], s["scales8"]), weight)


# ---- what a pass cannot do without -------------------------------------------------------------


def work(case):
    m, n, k = case["m"], case["n"], case["k"]
    held = m * k + m * k // GROUP  # rows in 8 bits
    if case["kind"] == "norm":
        # x, residual and weight in; the sum and the rows out.
        return dict(bytes=6 * m * k + 2 * k + held, flops=8 * m * k)
    rows = 2 * n if "glu" in case["kind"] else n
    moved = rows * k // 2 + rows * k // GROUP + 2 * m * n
    return dict(bytes=moved + (held if case["kind"] == "rows glu" else 2 * m * k), flops=2 * m * rows * k)


# ---- the same in 64 bits -----------------------------------------------------------------------


def _exact_scales(groups: torch.Tensor, most: float) -> torch.Tensor:
    """groups (..., 32) in 64 bits to their powers of two (...)."""
    top = groups.abs().amax(-1) / most
    scale = torch.exp2(torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -130))))
    scale = torch.where(top > scale, 2 * scale, torch.where(top <= scale / 2, scale / 2, scale))
    return torch.clamp(scale, min=2.0 ** -126)


def _e4m3(x: torch.Tensor) -> torch.Tensor:
    """x (64 bits, within 448) to the nearest e4m3 value, ties to even: steps of 2^(e - 3), e at least -6."""
    _, e = torch.frexp(x)
    step = torch.exp2(torch.clamp(e - 1, min=-6).double() - 3)
    return torch.round(x / step) * step


def _exact_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    groups = x.double().unflatten(-1, (-1, GROUP))
    scale = _exact_scales(groups, 448.0)
    return _e4m3(groups / scale[..., None]).flatten(-2), scale


def _exact_weight(s, first: int, rows: int) -> torch.Tensor:
    """Packed rows first .. first + rows - 1 of the 4-bit weight: (rows, K)."""
    k = s["case"]["k"]
    n = torch.arange(first, first + rows, device="cuda")[:, None]
    at = torch.arange(k, device="cuda")[None]
    byte = s["codes"][n // 16, at // 128, 16 * (at % 128 // 32 * 16 + n % 16) + at % 32 // 2].int()
    code = torch.where(at % 2 == 1, byte >> 4, byte & 15)
    kind, low = code >> 1 & 3, (code & 1).double()  # the two exponent bits, the mantissa bit
    size = torch.where(kind == 0, 0.5 * low, torch.exp2(kind.double() - 1) * (1 + 0.5 * low))
    e = s["scales"].view(torch.uint8)[n // 16, at // 512, 4 * (at % 128 // 32 * 16 + n % 16) + at % 512 // 128]
    return torch.where(code > 7, -size, size) * torch.exp2(e.double() - 127)


def exact(case, seed):
    s = prepare(case, seed)
    m, n, kind = case["m"], case["n"], case["kind"]
    if kind == "norm":
        hidden = s["x"].double() + s["residual"].double()
        h = hidden.to(torch.bfloat16).double()
        normed = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)).to(torch.bfloat16).double()
        return hidden, *_exact_rows((normed * s["weight"].double()).to(torch.bfloat16))
    if kind == "rows glu":
        x = s["codes8"].double().unflatten(-1, (-1, GROUP))
        x = (x * torch.exp2(s["scales8"].view(torch.uint8).double() - 127)[..., None]).flatten(-2)
    elif kind == "rows linear":
        codes, scale = _exact_rows(s["x"])
        x = (codes.unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)
    else:
        x = s["x"].double()
    out = torch.empty(m, n, dtype=torch.float64, device="cuda")
    for a in range(0, n, 1024):  # columns of the output, 1024 at a time
        b = min(a + 1024, n)
        if "glu" not in kind:
            out[:, a:b] = x @ _exact_weight(s, a, b - a).t()
            continue
        tiles = _exact_weight(s, 2 * a, 32 * ((b - a + 15) // 16)).view(-1, 2, 16, case["k"])
        gate, up = (x @ tiles[:, which].reshape(-1, case["k"])[:b - a].t() for which in (0, 1))
        out[:, a:b] = gate * torch.sigmoid(gate) * up
    return out
