"""4-bit weights of no rows, and calls of no token rows, through the operators on the GPU."""

from __future__ import annotations

import pytest
import torch

from fp4_helpers import activations, random_weight, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(0, 40), (5, 0), (0, 0)])
def test_products(pkg, m, n):
    ops = pkg.ops
    x = activations(m, 544, 1).cuda()
    rows = ops.quantize_rows_fp8(x)
    assert rows.codes.shape == (m, 544) and rows.scales.shape == (m, 17)
    for glu in (False, True):
        w = weight(pkg, *random_weight((1 + glu) * n, 544, 2), glu)
        assert (w.n, w.k) == (n, 544)
        assert (ops.w4a16_glu if glu else ops.w4a16_linear)(x, w).shape == (m, n)
        assert (ops.w4a8_glu if glu else ops.w4a8_linear)(rows, w).shape == (m, n)
        codes, scales = ops.unpack_fp4(w)
        assert ops.dequantize_fp4(codes, scales).shape == ((1 + glu) * n, 544)


def test_quantizers(pkg):
    ops = pkg.ops
    for n, k in ((0, 64), (3, 0)):
        codes, scales = ops.quantize_weight_fp4(torch.zeros(n, k, device="cuda"))
        assert codes.shape == (n, k // 2) and scales.shape == (n, k // 32)
    rows = ops.quantize_rows_fp8(torch.zeros(3, 0, dtype=torch.bfloat16, device="cuda"))
    assert rows.codes.shape == rows.scales.shape == (3, 0)
    with pytest.raises(RuntimeError, match="K > 0"):
        ops.w4a8_linear(rows, weight(pkg, *random_weight(16, 0, 1)))
