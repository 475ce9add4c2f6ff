"""4-bit weights and rows in 8 bits from their definitions, in 64 bits on the CPU: what the tests hold the kernels to.

A group is 32 consecutive k of a row. Its scale is the smallest power of two s >= 2^-126 with |v| <= top * s for every
finite v (top: 6 for weights, 448 for rows), as an e8m0 byte b = log2(s) + 127. Weights go to the nearest e2m1
value of w / s, ties to the even code, and a group that holds infinity or NaN gets the byte 255 (NaN); row values go to
the nearest e4m3 value of v / s, ties to even, but to none that stands for 2^128, and infinity and NaN to NaN.
"""

from __future__ import annotations

import torch

GROUP = 32
FP4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def scale_bytes(groups: torch.Tensor, top: float) -> torch.Tensor:
    """groups (..., 32) in 64 bits → bytes (...)."""
    amax = torch.where(torch.isfinite(groups), groups.abs(), 0.0).amax(-1)
    powers = torch.exp2(torch.arange(-126, 128, dtype=torch.float64, device=groups.device)) * top
    return torch.searchsorted(powers, amax.contiguous()) + 1  # the first power with amax <= it; byte 1 is 2^-126


def power(byte: torch.Tensor) -> torch.Tensor:
    """2^(byte - 127) in 64 bits, NaN for 255."""
    return torch.where(byte == 255, float("nan"), torch.exp2(byte.double() - 127))


def quantize_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """w (N, K) → e2m1 codes (N, K), one a byte, and scale bytes (N, K / 32)."""
    groups = w.double().unflatten(-1, (-1, GROUP))
    byte = torch.where(torch.isfinite(groups).all(-1), scale_bytes(groups, 6.0), 255)
    v = (groups / torch.where(byte == 255, 1.0, torch.exp2(byte.double() - 127))[..., None]).flatten(-2)
    away = (v.abs()[..., None] - FP4).abs()
    best = away.amin(-1, keepdim=True)
    # Among equally near values the even code.
    even = torch.where(away == best, torch.arange(8) % 2 * 100 + torch.arange(8), 1000)
    code = torch.where(torch.isfinite(v), even.argmin(-1), 0)
    top = (byte == 253).repeat_interleave(GROUP, -1)  # 2^126: codes 6 and 7 stand for 2^128 and more
    code = torch.where(top & (code > 5), 5, code)
    code = torch.where((v < 0) & (code > 0), code + 8, code)
    code = torch.where((byte == 255).repeat_interleave(GROUP, -1), 0, code)
    return code, byte


def weight_values(code: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    value = torch.where(code >= 8, -FP4[code % 8], FP4[code % 8])
    return value * power(byte).repeat_interleave(GROUP, -1)


def two_a_byte(code: torch.Tensor) -> torch.Tensor:
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8)


def tiles(code: torch.Tensor, byte: torch.Tensor, glu: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """The tile layout, byte by byte: codes (tiles, ceil(K / 128), 1024), scales (tiles, ceil(K / 512), 256)."""
    rows, k = code.shape
    n = rows // 2 if glu else rows
    count = -(-n // 16) * (2 if glu else 1)
    out = torch.zeros(count, -(-k // 128), 1024, dtype=torch.uint8)
    sout = torch.full((count, -(-k // 512), 256), 127, dtype=torch.uint8)
    for rb in range(count):
        for r in range(16):
            inner = 16 * (rb // 2 if glu else rb) + r
            if inner >= n:
                continue
            row = inner + (rb % 2) * n if glu else inner
            for b in range(k // GROUP):  # a group of the row
                j, g = b // 4, b % 4
                lane = 16 * g + r
                out[rb, j, 16 * lane:16 * lane + 16] = two_a_byte(code[row, 32 * b:32 * b + 32])
                sout[rb, j // 4, 4 * lane + j % 4] = byte[row, b]
    return out, sout


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """v within 448 (64 bits) to the nearest e4m3 value, ties to even: steps of 2^(e - 3), e at least -6."""
    _, e = torch.frexp(v)
    step = torch.exp2(torch.clamp(e - 1, min=-6).double() - 3)
    return torch.round(v / step) * step


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (M, K) → the e4m3 codes' values (M, K) in 64 bits and scale bytes (M, K / 32)."""
    groups = x.double().unflatten(-1, (-1, GROUP))
    byte = scale_bytes(groups, 448.0)
    scale = torch.exp2(byte.double() - 127)[..., None]
    finite = torch.isfinite(groups)
    v = e4m3(torch.where(finite, groups, 0.0) / scale)
    most = 2.0 ** 128 / scale
    below = e4m3(most * (1 - 2.0 ** -5))  # the largest value under 2^128 / scale where that is an e4m3 value
    v = torch.where(v.abs() >= most, torch.sign(v) * below, v)
    return torch.where(finite, v, float("nan")).flatten(-2), byte


def row_values(v: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    return v * power(byte).repeat_interleave(GROUP, -1)


def product(x: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(sum_k x w, sum_k |x w|), both (M, N) in 64 bits."""
    return x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()


def glu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    return gate * torch.sigmoid(gate) * up


def add_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float):
    """(s, n): s = bf16(x + residual), n = bf16(w bf16(fp32(s / sqrt(mean(s^2) + eps)))), both bf16."""
    s = x if residual is None else (x.double() + residual.double()).to(torch.bfloat16)
    h = s.double()
    t = (h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)).float().to(torch.bfloat16)
    return s, (weight.double() * t.double()).to(torch.bfloat16)
