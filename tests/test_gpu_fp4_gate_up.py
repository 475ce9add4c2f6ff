"""`Fp4GateUp`, by itself and in the MLP and the decode runner, against silu(x G^T) (x U^T) in 64 bits, G and U the gate
and up weights as the oracle quantizes them. Bounds as in test_gpu_fp4_gemm.py."""

from __future__ import annotations

import pytest
import torch

from fp4_helpers import activations
from oracle import fp4 as ora
from test_gpu_fp4_gemm import _glu_bound, _values
from test_gpu_fp4_modules import MODES, _linear, _near, _runner

pytestmark = pytest.mark.gpu


def _check(h, x, gate, up, mode):
    """h against the definition over bf16 rows x and bf16 weights."""
    rows = mode == "w4a8"
    g64, u64 = (ora.weight_values(*ora.quantize_weight(t.detach().cpu())).cuda() for t in (gate, up))
    values = _values(x.reshape(-1, x.shape[-1]).cpu(), rows).cuda()
    (g, sg), (u, su) = ora.product(values, g64), ora.product(values, u64)
    off = (h.reshape(g.shape).double() - ora.glu(g, u)).abs()
    bound = _glu_bound(g, sg, u, su, x.shape[-1], rows)
    assert bool((off <= bound).all()), float((off / bound).max())
    # Gate and up are not alike: the other way round is not within the bounds.
    swapped = (h.reshape(g.shape).double() - ora.glu(u, g)).abs()
    assert bool((swapped > _glu_bound(u, su, g, sg, x.shape[-1], rows)).any())


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("m,n,k", [(1, 320, 256), (20, 330, 544), (64, 1056, 512), (300, 1500, 288)])
def test_module(pkg, mode, m, n, k):
    gate, up = _linear(n, k, 3), _linear(n, k, 4)
    mod = pkg.Fp4GateUp.from_linears(gate, up, mode)
    x = activations(m, k, m).cuda()
    h = mod(x)
    assert h.shape == (m, n)
    _check(h, x, gate.weight, up.weight, mode)
    values = torch.cat([ora.weight_values(*ora.quantize_weight(t.weight.detach().cpu())) for t in (gate, up)])
    assert torch.equal(mod.dequantized().double().cpu(), values)


@pytest.mark.parametrize("mode", MODES)
def test_mlp(pkg, mode):
    from transformers import LlamaConfig
    from transformers.models.llama.modeling_llama import LlamaMLP

    torch.manual_seed(5)
    mlp = LlamaMLP(LlamaConfig(hidden_size=256, intermediate_size=416)).to("cuda", torch.bfloat16)
    mod = pkg.Fp4GluMLP.from_mlp(mlp, mode)
    x = activations(30, 256, 6).cuda().view(2, 15, 256)
    h = mod.gate_up(x)
    _check(h, x, mlp.gate_proj.weight, mlp.up_proj.weight, mode)
    down = ora.weight_values(*ora.quantize_weight(mlp.down_proj.weight.detach().cpu())).cuda()
    _near(mod(x), h, down, mode)


@pytest.mark.parametrize("mode", MODES)
def test_decode_runner(pkg, mode):
    """Gate and up of a prompt and a step, on the very input that they saw."""
    runner = _runner(pkg)
    runner.quantize(mode)
    runner.use("fp4")
    seen, calls = runner._lin, []

    def checked(i, name, x):
        y = seen(i, name, x)
        if name == "gate_up":
            bf16 = x if isinstance(x, torch.Tensor) else pkg.ops.dequantize_rows_fp8(pkg.ops.Fp8Rows(x.xq, x.sx))
            mlp = runner.layers[i].mlp
            _check(y, bf16, mlp.gate_proj.weight, mlp.up_proj.weight, mode)
            calls.append(i)
        return y

    runner._lin = checked
    tokens = torch.randint(0, 300, (5, 20), generator=torch.Generator().manual_seed(1)).cuda()
    runner.prefill(tokens)
    runner.step(tokens[:, 0], 20)
    assert calls == [0, 1, 0, 1]
