"""What makes the operands of the 4-bit products on the GPU, bit for bit against the definitions in 64 bits."""

from __future__ import annotations

import pytest
import torch

from fp4_helpers import E8, F8, activations
from oracle import fp4 as ora

pytestmark = pytest.mark.gpu


def _bytes(t):
    return t.view(torch.uint8).cpu()


def _weights(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(n, k, generator=g) * torch.exp(2 * torch.randn(n, 1, generator=g))
    w[0] = 0.0
    # Ties between neighbouring codes, and values at the edge between two scales.
    edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.0001, 5.9999, -0.25, -0.75, -5.0, 3.0, -0.0, 1e-9])
    w[-1, :16] = edge
    if n > 2:
        w[1, :32] = torch.linspace(-6, 6, 32) * 2.0 ** -125
        w[2, :32] = torch.linspace(-1, 1, 32) * 3.4e38
    return w


@pytest.mark.parametrize("n,k", [(1, 32), (17, 96), (40, 544), (300, 2080)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_weight_quantizer(pkg, n, k, dtype):
    w = _weights(n, k, n)
    w = (w.clamp(-60000, 60000) if dtype is torch.float16 else w).to(dtype)
    codes, scales = pkg.ops.quantize_weight_fp4(w.cuda())
    code, byte = ora.quantize_weight(w)
    assert torch.equal(_bytes(scales), byte.to(torch.uint8))
    assert torch.equal(codes.cpu(), ora.two_a_byte(code))
    values, want = pkg.ops.dequantize_fp4(codes, scales).double().cpu(), ora.weight_values(code, byte)
    # In bf16 and fp16 the largest weights are infinities: their groups are NaN.
    assert torch.equal(torch.isnan(values), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(values), torch.nan_to_num(want))


def test_weight_groups_that_are_not_finite(pkg):
    w = torch.ones(3, 96)
    w[0, 5], w[1, 40], w[2, 95] = float("inf"), float("nan"), -float("inf")
    _, scales = pkg.ops.quantize_weight_fp4(w.cuda())
    nan = _bytes(scales) == 255
    assert nan.tolist() == [[True, False, False], [False, True, False], [False, False, True]]


def test_weight_quantizer_takes_a_strided_weight(pkg):
    w = _weights(40, 640, 3)
    both = [pkg.ops.quantize_weight_fp4(t) for t in (w.cuda()[:, 32:].contiguous(), w.cuda()[:, 32:], )]
    assert all(torch.equal(_bytes(a), _bytes(b)) for a, b in zip(*both))


@pytest.mark.parametrize("glu", [False, True])
@pytest.mark.parametrize("n,k", [(2, 32), (32, 128), (34, 512), (70, 1184), (48, 544)])
def test_tiles(pkg, n, k, glu):
    g = torch.Generator().manual_seed(n)
    code, byte = torch.randint(0, 16, (n, k), generator=g), torch.randint(1, 255, (n, k // 32), generator=g)
    codes, scales = ora.two_a_byte(code).cuda(), byte.to(torch.uint8).view(E8).cuda()
    w = pkg.ops.pack_fp4(codes, scales, glu)
    want = ora.tiles(code, byte, glu)
    assert (w.n, w.k) == (n // 2 if glu else n, k)
    assert torch.equal(w.codes.cpu(), want[0]) and torch.equal(_bytes(w.scales), want[1])
    back = pkg.ops.unpack_fp4(w)
    assert torch.equal(back[0], codes) and torch.equal(_bytes(back[1]), _bytes(scales))


def _rows(m, k, seed):
    x = activations(m, k, seed)
    x[0, :32] = 0
    x[-1, -32:] = torch.tensor([448.0, 450.0, -448.0, 0.0078125] * 8) * 2.0 ** -3
    if m > 2:
        x[1, :32] = torch.linspace(-3e38, 3e38, 32).to(torch.bfloat16)
        x[1, 32:64] = torch.linspace(-1e-38, 1e-38, 32).to(torch.bfloat16)
        x[2, 3], x[2, 40], x[2, 41] = float("inf"), float("nan"), -float("inf")
    return x


def _same_rows(rows, v, byte):
    assert rows.codes.dtype == F8 and rows.scales.dtype == E8
    assert torch.equal(_bytes(rows.scales), byte.to(torch.uint8).view(rows.scales.shape))
    got = rows.codes.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(v).view(got.shape))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(v).view(got.shape))


@pytest.mark.parametrize("m,k", [(1, 32), (3, 64), (5, 4096), (33, 1184), (300, 14336)])
def test_rows(pkg, m, k):
    x = _rows(m, k, m) if k >= 64 else activations(m, k, m)
    _same_rows(pkg.ops.quantize_rows_fp8(x.cuda()), *ora.quantize_rows(x))


def test_rows_keep_their_shape_and_take_strides(pkg):
    x = activations(6, 320, 1).cuda().view(2, 3, 320)
    rows = pkg.ops.quantize_rows_fp8(x)
    assert rows.codes.shape == (2, 3, 320) and rows.scales.shape == (2, 3, 10)
    for part in (x[..., 32:], x[..., 1:289], x.transpose(0, 1), x[:, 1]):
        _same_rows(pkg.ops.quantize_rows_fp8(part), *ora.quantize_rows(part.cpu().reshape(-1, part.shape[-1])))
    empty = pkg.ops.quantize_rows_fp8(x[:0])
    assert empty.codes.shape == (0, 3, 320)


@pytest.mark.parametrize("m,k", [(1, 32), (3, 96), (33, 4096), (64, 4128), (5, 8224), (2, 16384)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(pkg, m, k, residual):
    """The bits of the formula in 64 bits: r is off by 2^-40 of itself, which puts s r at another fp32 value once in 2^16
    values, and that at another bf16 one once in 2^32."""
    x, r = activations(m, k, 1).cuda(), activations(m, k, 2).cuda()
    w = (0.5 + torch.rand(k, generator=torch.Generator().manual_seed(3))).to(torch.bfloat16).cuda()
    s, rows = pkg.ops.add_rmsnorm_fp8(x, r if residual else None, w, 1e-5)
    s64, n64 = ora.add_norm(x.cpu(), r.cpu() if residual else None, w.cpu(), 1e-5)
    assert torch.equal(s.cpu(), s64)
    _same_rows(rows, *ora.quantize_rows(n64))
    s2, normed = pkg.ops.add_rmsnorm(x, r if residual else None, w, 1e-5)
    assert torch.equal(s, s2)
    # Two roundings of half a bf16 step each on both sides, at most two steps apart after the weight's product.
    off = (normed.cpu().double() - n64.double()).abs()
    assert bool((off <= 2.0 ** -6 * n64.double().abs()).all()) and float((off > 0).double().mean()) < 1e-3


@pytest.mark.parametrize("m,k", [(3700, 4096), (1900, 8000), (900, 16384)])
def test_norm_of_large_calls(pkg, m, k):
    """More than 96 MiB of traffic, to the bit."""
    assert 7 * m * k > 96 << 20
    x, r, w = activations(m, k, 1).cuda(), activations(m, k, 2).cuda(), activations(1, k, 3)[0].cuda()
    s, rows = pkg.ops.add_rmsnorm_fp8(x, r, w, 1e-5)
    s64, n64 = ora.add_norm(x, r, w, 1e-5)
    assert torch.equal(s, s64)
    for at in range(0, m, 500):
        _same_rows(pkg.ops.Fp8Rows(*(t[at:at + 500] for t in rows)), *(t.cpu() for t in ora.quantize_rows(n64[at:at + 500])))


@pytest.mark.parametrize("scale", [1e-25, 1e-10, 1e10, 1e25])
def test_norm_of_very_large_and_small_rows(pkg, scale):
    """Squares past fp32's range, and no eps that would hide them; a row of zeros has no norm then."""
    x = (activations(5, 512, 8).double() * scale).to(torch.bfloat16)
    x[3] = 0
    w = activations(1, 512, 9)[0]
    _, rows = pkg.ops.add_rmsnorm_fp8(x.cuda(), None, w.cuda(), 0.0)
    _same_rows(rows, *ora.quantize_rows(ora.add_norm(x, None, w, 0.0)[1]))
    assert bool(torch.isnan(rows.codes[3].float()).all())


def test_norm_of_rows_that_are_not_finite(pkg):
    x = activations(4, 256, 5)
    x[1, 7], x[2, 9] = float("inf"), float("nan")
    w = torch.ones(256, dtype=torch.bfloat16)
    _, rows = pkg.ops.add_rmsnorm_fp8(x.cuda(), None, w.cuda(), 1e-5)
    _same_rows(rows, *ora.quantize_rows(ora.add_norm(x, None, w, 1e-5)[1]))
    assert not bool(torch.isnan(rows.codes[0].float()).any()) and not bool(torch.isnan(rows.codes[3].float()).any())
