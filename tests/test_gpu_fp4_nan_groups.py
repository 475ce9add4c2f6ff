"""Groups that are not finite: the weight quantizer gives them the scale NaN and codes of zero, and every output that such
a group is part of is NaN, whatever the rows hold; the others' bits stay."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from fp4_choice import choice
from fp4_helpers import E8, activations

pytestmark = pytest.mark.gpu

# M, N, K: the kernel for few rows at each of its widths, and every tile.
SIZES = [(1, 40, 640), (7, 300, 544), (40, 3600, 544), (40, 14330, 160), (777, 1500, 288), (300, 8190, 160), (777, 6150, 96),
         (260, 2050, 14400)]


def _weight(n, k, bad, seed):
    """A weight with values that are not finite at bad: ((row, k), ...)."""
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) * 2.0 ** -5
    whole = w.clone()
    for i, (row, at) in enumerate(bad):
        w[row, at] = (float("inf"), float("nan"), -float("inf"))[i % 3]
        whole[row, at // 32 * 32:at // 32 * 32 + 32] = 0
    return w, whole


def test_the_sizes_reach_every_kernel(pkg):
    assert {choice(pkg, m, n, k, False, False)[:2] for m, n, k in SIZES} >= {(32, 128), (64, 128), (64, 256)}
    assert {choice(pkg, m, n, k, True, False)[:2] for m, n, k in SIZES} >= {(32, 128), (64, 128), (128, 256)}


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(pkg, m, n, k, rows):
    ops = pkg.ops
    bad = [(0, 0), (n // 2, k - 1), (n - 1, k // 2)]
    w, whole = (ops.pack_fp4(*ops.quantize_weight_fp4(t.cuda())) for t in _weight(n, k, bad, m))
    x = activations(m, k, m).cuda()
    x[m // 2] = 0  # NaN times zero
    x = ops.quantize_rows_fp8(x) if rows else x
    linear = ops.w4a8_linear if rows else ops.w4a16_linear
    y, want = linear(x, w), linear(x, whole)
    nan = torch.zeros(n, dtype=torch.bool, device="cuda")
    nan[[row for row, _ in bad]] = True
    assert bool(torch.isnan(y[:, nan].float()).all())
    assert torch.equal(y[:, ~nan], want[:, ~nan])


@pytest.mark.parametrize("rows", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("m,n,k", [(1, 40, 640), (33, 6150, 96), (70, 6150, 160), (777, 1500, 288), (300, 8190, 160)])
def test_glu(pkg, m, n, k, rows):
    ops = pkg.ops
    bad = [(0, 0), (n // 2, k - 1), (n + 5, k // 2)]  # two columns of gate and one of up
    w, whole = (ops.pack_fp4(*ops.quantize_weight_fp4(t.cuda()), glu=True) for t in _weight(2 * n, k, bad, m))
    x = activations(m, k, m).cuda()
    x = ops.quantize_rows_fp8(x) if rows else x
    glu = ops.w4a8_glu if rows else ops.w4a16_glu
    y, want = glu(x, w), glu(x, whole)
    nan = torch.zeros(n, dtype=torch.bool, device="cuda")
    nan[[row % n for row, _ in bad]] = True
    assert bool(torch.isnan(y[:, nan].float()).all())
    assert torch.equal(y[:, ~nan], want[:, ~nan])


@pytest.mark.parametrize("m,n,k", SIZES)
def test_rows_with_a_scale_of_nan(pkg, m, n, k):
    """Rows in 8 bits whose group has the scale NaN over codes of zero."""
    ops = pkg.ops
    w = ops.pack_fp4(*ops.quantize_weight_fp4(_weight(n, k, [], m)[0].cuda()))
    held = ops.quantize_rows_fp8(activations(m, k, m).cuda())
    want = ops.w4a8_linear(held, w)
    codes, scales = held.codes.clone(), held.scales.view(torch.uint8).clone()
    codes.view(torch.uint8)[m // 2, k - 32:] = 0
    scales[m // 2, k // 32 - 1] = 255
    y = ops.w4a8_linear(ops.Fp8Rows(codes, scales.view(E8)), w)
    others = torch.arange(m, device="cuda") != m // 2
    assert bool(torch.isnan(y[m // 2].float()).all()) and torch.equal(y[others], want[others])


@pytest.mark.parametrize("mode", ["w4a16", "w4a8"])
def test_module(pkg, mode):
    lin = nn.Linear(256, 40, bias=False, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        lin.weight[7, 100] = float("nan")
    mod = pkg.Fp4Linear.from_linear(lin, mode)
    y = mod(activations(3, 256, 1).cuda())
    assert bool(torch.isnan(y[:, 7].float()).all()) and int(torch.isnan(y.float()).sum()) == 3
    assert bool(torch.isnan(mod.dequantized()[7, 96:128]).all())
