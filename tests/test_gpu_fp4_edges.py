"""Calls of the 4-bit products and of what makes their rows that the sizes of the other tests do not make: K split over
workgroups, values that are not finite, strides and paddings, the smallest and largest scales, offsets past 32 bits."""

from __future__ import annotations

import pytest
import torch

from fp4_helpers import E8, F8, activations, random_weight, weight
from oracle import fp4 as ora
from test_gpu_fp4_gemm import _bound, _check

pytestmark = pytest.mark.gpu

KINDS = [(1, 40, 640), (13, 100, 1184), (40, 3600, 544), (100, 64, 96), (300, 500, 1056), (700, 1100, 640),
         (1050, 6100, 544)]


SPLIT = [(300, 1030, 14336, False), (260, 2050, 14400, False), (130, 530, 28704, True)]  # K over 2 to 8 workgroups


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k,glu", [(200, 1030, 14336, False), (40, 4096, 14368, False), (200, 512, 14400, True), *SPLIT])
def test_split_k(pkg, m, n, k, glu, rows):
    from llm_serving_engine_amd import _lib

    args = _lib.FP4_GEMM_ARGS.pack(16, k, 16 if rows else 0, k // 32 + 3 & ~3, 16, 16, 16, n, m, n, k, int(glu))
    if (m, n, k, glu) in SPLIT:
        assert pkg.library().lse_fp4_gemm_workspace_bytes(args) > 0
    _check(pkg, m, n, k, rows, glu, seed=m)


def _product(pkg, x, w, rows):
    return pkg.ops.w4a8_linear(pkg.ops.quantize_rows_fp8(x), w) if rows else pkg.ops.w4a16_linear(x, w)


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", KINDS)
def test_rows_do_not_reach_each_other(pkg, m, n, k, rows):
    """A row with infinity or NaN makes its own outputs so, and the other rows' bits stay; so do those of a permuted
    call. A group of the weight with the scale NaN reaches its own column alone."""
    code, byte = random_weight(n, k, m)
    w = weight(pkg, code, byte)
    x = activations(m, k, m).cuda()
    y = _product(pkg, x, w, rows)
    perm = torch.randperm(m, generator=torch.Generator().manual_seed(1)).cuda()
    assert torch.equal(_product(pkg, x[perm], w, rows), y[perm])
    bad = x.clone()
    bad[m // 2, k - 1] = float("nan")
    z = _product(pkg, bad, w, rows)
    others = torch.arange(m, device="cuda") != m // 2
    assert torch.equal(z[others], y[others])
    touched = (code[:, k - 1] >= 0).cuda()
    assert bool(torch.isnan(z[m // 2][touched].float()).all())
    if not rows:  # rows in 8 bits hold infinity as NaN
        bad[m // 2, k - 1] = float("inf")
        z = _product(pkg, bad, w, rows)
        assert torch.equal(z[others], y[others])
        value = ora.weight_values(code, byte)[:, k - 1].cuda()
        want = torch.where(value == 0, float("nan"), torch.sign(value) * float("inf"))
        assert torch.equal(torch.nan_to_num(z[m // 2].double(), nan=7.0), torch.nan_to_num(want, nan=7.0))
    byte[n // 3, k // 32 - 1] = 255
    z = _product(pkg, x, weight(pkg, code, byte), rows)
    columns = torch.arange(n, device="cuda") != n // 3
    assert torch.equal(z[:, columns], y[:, columns]) and bool(torch.isnan(z[:, n // 3].float()).all())


@pytest.mark.parametrize("m,n,k", KINDS)
def test_strided_rows(pkg, m, n, k):
    """Rows in 8 bits out of wider tensors: codes at strides and offsets that kernels take and that they do not, scales at
    every stride, with NaN scales behind each row."""
    code, byte = random_weight(n, k, m)
    w = weight(pkg, code, byte)
    ops, per = pkg.ops, k // 32
    rows = ops.quantize_rows_fp8(activations(m, k, 3).cuda())
    want = ops.w4a8_linear(rows, w)
    for pad, first, spad, sfirst in ((32, 16, 8, 4), (16, 0, 1, 0), (24, 8, 3, 1), (48, 32, 4 - per % 4, 0)):
        codes = torch.full((m, k + pad), 0x7f, dtype=torch.uint8, device="cuda").view(F8)
        codes[:, first:first + k] = rows.codes
        scales = torch.full((m, per + spad), 255, dtype=torch.uint8, device="cuda")
        scales[:, sfirst:sfirst + per] = rows.scales.view(torch.uint8)
        part = ops.Fp8Rows(codes[:, first:first + k], scales.view(E8)[:, sfirst:sfirst + per])
        assert torch.equal(ops.w4a8_linear(part, w), want)
    exact = ops.Fp8Rows(rows.codes.clone(), rows.scales.contiguous().clone())
    assert torch.equal(ops.w4a8_linear(exact, w), want)
    if m % 2 == 0:
        folded = ops.Fp8Rows(rows.codes.view(2, m // 2, k), rows.scales.reshape(2, m // 2, per))
        assert torch.equal(ops.w4a8_linear(folded, w), want.view(2, m // 2, n))


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", KINDS)
def test_outputs_stay_in_their_columns(pkg, m, n, k, rows):
    """With a row stride past N, at every alignment: what lies between and behind the rows stays."""
    from llm_serving_engine_amd import _lib

    code, byte = random_weight(n, k, m)
    w = weight(pkg, code, byte)
    x = activations(m, k, 4).cuda()
    want = _product(pkg, x, w, rows)
    held = pkg.ops.quantize_rows_fp8(x) if rows else None
    for extra, shift in ((1, 0), (3, 1), (4, 2), (8, 4)):
        y = torch.full((m + 2, n + extra), 3.0, dtype=torch.bfloat16, device="cuda")
        at = y.data_ptr() + 2 * shift
        scales = (held.scales.data_ptr(), held.scales.stride(0) if m > 1 else k // 32 + 3 & ~3) if rows else (0, 0)
        args = _lib.FP4_GEMM_ARGS.pack(held.codes.data_ptr() if rows else x.data_ptr(), k, *scales, w.codes.data_ptr(),
                                       w.scales.data_ptr(), at, n + extra, m, n, k, 0)
        pkg.ops._launch(0, "lse_fp4_gemm", args, None, 0)
        flat = y.view(-1)[shift:shift + m * (n + extra)].view(m, n + extra)
        assert torch.equal(flat[:, :n], want)
        flat[:, :n] = 3.0
        assert bool((y == 3.0).all())


def test_scales_at_their_ends(pkg):
    """The smallest weights against the largest rows and the other way: products are exact as long as they and the weight
    are normal numbers."""
    k = 256
    code = torch.randint(0, 16, (48, k), generator=torch.Generator().manual_seed(1))
    for wb, size in ((2, 100.0), (3, 90.0), (250, -100.0), (252, -110.0)):
        byte = torch.full((48, k // 32), wb)
        w = weight(pkg, code, byte)
        x = torch.zeros(5, k)
        x[torch.arange(5), torch.tensor([0, 40, 100, 200, 255])] = 2.0 ** size
        want = x.double() @ ora.weight_values(code, byte).t()
        assert torch.equal(pkg.ops.w4a16_linear(x.bfloat16().cuda(), w).double().cpu(), want)
        held = pkg.ops.quantize_rows_fp8(x.bfloat16().cuda())
        assert torch.equal(pkg.ops.w4a8_linear(held, w).double().cpu(), want)


def test_a_stride_past_the_kernels(pkg):
    """Rows further apart than 32-bit offsets allow are gathered first."""
    code, byte = random_weight(32, 64, 5)
    w = weight(pkg, code, byte)
    base = torch.zeros(4 * (3 << 20), dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((4, 64), (3 << 20, 1))
    x.copy_(activations(4, 64, 6))
    assert torch.equal(pkg.ops.w4a16_linear(x, w), pkg.ops.w4a16_linear(x.contiguous(), w))


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
def test_outputs_past_32_bits(pkg, rows):
    """2.3e9 outputs: the last rows and columns are where they belong."""
    m, n, k = 70000, 32768, 32
    code, byte = random_weight(n, k, 7)
    x = torch.zeros(m, k, dtype=torch.bfloat16)
    x[-300:] = activations(300, k, 8)
    y = _product(pkg, x.cuda(), weight(pkg, code, byte), rows)
    values = (ora.row_values(*ora.quantize_rows(x[-300:])) if rows else x[-300:].double()).cuda()
    want, s = ora.product(values, ora.weight_values(code, byte).cuda())
    assert bool(((y[-300:].double() - want).abs() <= _bound(want, s, k, rows)).all())
    assert not bool(y[0].any()) and not bool(y[m // 2].any())


def test_rows_past_32_bits(pkg):
    """2.3e9 values through the quantizer and the norm."""
    m, k = 140000, 16384
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-2:] = activations(2, k, 9).cuda()
    w = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    few = pkg.ops.quantize_rows_fp8(x[-2:])
    all_ = pkg.ops.quantize_rows_fp8(x)
    for a, b in zip(all_, few):
        assert torch.equal(a[-2:].view(torch.uint8), b.view(torch.uint8))
    del all_
    s, normed = pkg.ops.add_rmsnorm_fp8(x, x, w, 1e-5)
    s2, normed2 = pkg.ops.add_rmsnorm_fp8(x[-2:], x[-2:], w, 1e-5)
    assert torch.equal(s[-2:], s2)
    for a, b in zip(normed, normed2):
        assert torch.equal(a[-2:].view(torch.uint8), b.view(torch.uint8))


def test_norm_of_strided_rows(pkg):
    x = activations(12, 640, 1).cuda()
    w = torch.linspace(0.5, 2, 257, device="cuda").bfloat16()[1:]  # at no multiple of 16 bytes
    for part, res in ((x[:, 32:288], x[:, 288:544]), (x[:, 3:259], x[:, 100:356]), (x[::2, :256], x[1::2, :256])):
        s, rows = pkg.ops.add_rmsnorm_fp8(part, res, w, 1e-6)
        s2, rows2 = pkg.ops.add_rmsnorm_fp8(part.contiguous(), res.contiguous(), w.clone(), 1e-6)
        assert torch.equal(s, s2)
        for a, b in zip(rows, rows2):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    s, rows = pkg.ops.add_rmsnorm_fp8(x.view(3, 4, 640), None, torch.ones(640, dtype=torch.bfloat16, device="cuda"), 1e-6)
    assert s.shape == rows.codes.shape == (3, 4, 640) and rows.scales.shape == (3, 4, 20)
    assert pkg.ops.add_rmsnorm_fp8(x[:0], None, torch.ones(640, dtype=torch.bfloat16, device="cuda"), 1e-6)[0].shape == (0, 640)
