"""Inputs of the 4-bit weight tests."""

from __future__ import annotations

import torch

from oracle import fp4 as ora

E8 = torch.float8_e8m0fnu
F8 = torch.float8_e4m3fn


def random_weight(n: int, k: int, seed: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (N, K), every one of the sixteen, and scale bytes (N, K / 32) of 2^-9 to 2^-5."""
    g = torch.Generator().manual_seed(seed)
    code = torch.randint(0, 16, (n, k), generator=g)
    return code, torch.randint(118, 123, (n, k // 32), generator=g)


def weight(pkg, code, byte, glu=False, dev="cuda"):
    """The weight in the product's tiles, packed on the GPU."""
    codes = ora.two_a_byte(code).to(dev)
    return pkg.ops.pack_fp4(codes, byte.to(torch.uint8).view(E8).to(dev), glu)


def activations(m: int, k: int, seed: int) -> torch.Tensor:
    """bf16 rows with some channels twenty times as large."""
    g = torch.Generator().manual_seed(seed)
    loud = 1.0 + 20.0 * (torch.rand(k, generator=g) < 0.01)
    return (torch.randn(m, k, generator=g) * loud).to(torch.bfloat16)


def rows8(pkg, x, dev="cuda"):
    return pkg.ops.quantize_rows_fp8(x.to(dev))


def few_ones(m: int, k: int, count: int, seed: int) -> torch.Tensor:
    """Rows of `count` values of 1 and -1 at random places, zeros elsewhere."""
    g = torch.Generator().manual_seed(seed)
    x = torch.zeros(m, k)
    at = torch.stack([torch.randperm(k, generator=g)[:count] for _ in range(m)])
    return x.scatter_(1, at, torch.randint(0, 2, at.shape, generator=g) * 2.0 - 1.0)
