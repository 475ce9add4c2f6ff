"""Modules over 4-bit weights, a model and a decode runner on them, and the operators one after another as such a model
runs them. Bounds as in test_gpu_fp4_gemm.py: 2^-8 |y| for the rounding, K 2^-24 S for fp32 sums, 2^-10 S for rows in 8
bits."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from fp4_helpers import activations, random_weight, weight
from oracle import fp4 as ora

pytestmark = pytest.mark.gpu

MODES = ["w4a16", "w4a8"]


def _linear(n, k, seed, bias=False):
    torch.manual_seed(seed)
    return nn.Linear(k, n, bias=bias, device="cuda", dtype=torch.bfloat16)


def _near(y, x, w, mode, bias=None):
    """y against x w^T in 64 bits (x rounded to 8 bits first in "w4a8")."""
    x = x.reshape(-1, x.shape[-1]).cpu()
    values = (ora.row_values(*ora.quantize_rows(x)) if mode == "w4a8" else x.double()).cuda()
    want, s = ora.product(values, w)
    bound = 2.0 ** -8 * want.abs() + s * (w.shape[1] * 2.0 ** -24 + (2.0 ** -10 if mode == "w4a8" else 0.0))
    if bias is not None:  # added to the rounded product, rounded again
        want = want + bias.double()
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
    off = (y.reshape(want.shape).double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_module(pkg, mode, bias):
    lin = _linear(200, 544, 1, bias)
    mod = pkg.Fp4Linear.from_linear(lin, mode)
    code, byte = ora.quantize_weight(lin.weight.detach().cpu())
    w = ora.weight_values(code, byte).cuda()
    assert torch.equal(mod.dequantized().double(), w)
    x = activations(30, 544, 2).cuda().view(2, 15, 544)
    y = mod(x)
    assert y.shape == (2, 15, 200)
    _near(y, x, w, mode, mod.bias)
    wide = torch.zeros(30, 1088, dtype=torch.bfloat16, device="cuda")
    wide[:, 64:608] = x.view(30, 544)
    assert torch.equal(mod(wide[:, 64:608]), y.view(30, 200))
    assert torch.equal(mod.to(torch.float32)(x.view(30, 544)) if not bias else y.view(30, 200), y.view(30, 200))
    assert mod(x[:0]).shape == (0, 15, 200)


@pytest.mark.parametrize("mode", MODES)
def test_mlp_and_norm_modules(pkg, mode):
    class Mlp(nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_proj, self.up_proj, self.down_proj = _linear(320, 256, 3), _linear(320, 256, 4), _linear(256, 320, 5)
            self.act_fn = nn.SiLU()

    class Norm(nn.Module):
        def __init__(self):
            super().__init__()
            self.weight = nn.Parameter(torch.linspace(0.5, 1.5, 256, device="cuda").bfloat16())
            self.variance_epsilon = 1e-5

    mod = pkg.Fp4GluMLP.from_mlp(Mlp(), mode)
    x = activations(20, 256, 6).cuda().view(4, 5, 256)
    if mode == "w4a8":
        norm = pkg.Fp8RMSNorm(Norm())
        rows = norm(x)
        assert rows.shape == x.shape and rows.dtype == torch.bfloat16 and rows.device == x.device
        _, normed = pkg.ops.add_rmsnorm(x, None, norm.weight, 1e-5)
        assert torch.equal(mod(rows), mod(normed))
        with pytest.raises(RuntimeError, match="reach a w4a16"):
            pkg.Fp4Linear.from_linear(_linear(32, 256, 7), "w4a16")(rows)
    h = mod.gate_up(x)
    assert torch.equal(mod.down_proj(h), mod(x))
    _near(mod(x), h, mod.down_proj.dequantized().double(), mode)


@pytest.mark.parametrize("mode", MODES)
def test_grouped_qkv_is_the_separate_products(pkg, mode):
    from llm_serving_engine_amd.fp4_linear import group_qkv_fp4

    attn = nn.Module()
    for i, (name, n) in enumerate((("q_proj", 256), ("k_proj", 64), ("v_proj", 64))):
        setattr(attn, name, pkg.Fp4Linear.from_linear(_linear(n, 512, i), mode))
    x = activations(7, 512, 9).cuda()
    apart = [getattr(attn, f"{n}_proj")(x).clone() for n in "qkv"]
    assert group_qkv_fp4(attn) is not None
    for _ in range(2):
        together = [getattr(attn, f"{n}_proj")(x) for n in "qkv"]
        assert all(torch.equal(a, b) for a, b in zip(apart, together))
    attn.to("cpu").to("cuda")  # the buffers are no views of the stack any more
    assert all(torch.equal(a, getattr(attn, f"{n}_proj")(x)) for a, n in zip(apart, "qkv"))


def _runner(pkg, batch=5, capacity=40):
    from llm_serving_engine_amd.decode_step import DecodeRunner, random_llama

    model = random_llama(2, 0, torch.device("cuda:0"), hidden_size=512, intermediate_size=1056, num_attention_heads=4,
                         num_key_value_heads=2, head_dim=128, vocab_size=300)
    return DecodeRunner(model, batch, capacity)


@pytest.mark.parametrize("cache", ["torch", "paged", "fp8"])
@pytest.mark.parametrize("mode", MODES)
def test_decode_runner(pkg, mode, cache):
    """Every projection of prompts and steps on the very input it saw, over each kind of K/V cache."""
    runner = _runner(pkg)
    runner.quantize(mode)
    runner.use("fp4")
    if cache == "paged":
        runner.enable_paged()
        runner.use_attention("paged")
    elif cache == "fp8":
        runner.enable_fp8_kv()
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 300, (5, 20), generator=g).cuda()
    runner.trace = []
    seen = runner._lin

    def checked(i, name, x):
        y = seen(i, name, x)
        mod = runner.fp4[i][name]
        if not isinstance(x, torch.Tensor):
            bf16 = pkg.ops.dequantize_rows_fp8(pkg.ops.Fp8Rows(x.xq, x.sx))
            assert mode == "w4a8" and name in ("qkv", "gate_up")
        else:
            assert mode == "w4a16" or name in ("o", "down")
            bf16 = x
        if name != "gate_up":
            _near(y, bf16, mod.dequantized().double(), mode)
        return y

    runner._lin = checked
    runner.prefill(tokens)
    logits = runner.step(tokens[:, 0], 20)
    assert logits.shape == (5, 300) and bool(torch.isfinite(logits.float()).all())


@pytest.mark.parametrize("mode", MODES)
def test_a_decode_step_replays_from_a_graph(pkg, mode):
    runner = _runner(pkg)
    runner.quantize(mode)
    runner.use("fp4")
    runner.enable_fp8_kv()
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 300, (5, 21), generator=g).cuda()
    runner.prefill(tokens[:, :20])
    step = tokens[:, 20].clone()
    want = runner.step(step, 20).clone()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        runner.step(step, 20)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = runner.step(step, 20)
    for i in range(4):
        other = torch.roll(tokens[:, 20], i)
        eager = runner.step(other, 20).clone()
        step.copy_(other)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        if i == 0:
            assert torch.equal(got, want)


@pytest.mark.parametrize("mode", MODES)
def test_quantized_llama(pkg, mode):
    """`quantize_model_` puts the modules in place, and the model runs on them."""
    from llm_serving_engine_amd.decode_step import random_llama

    model = random_llama(2, 3, torch.device("cuda:0"), hidden_size=256, intermediate_size=512, num_attention_heads=4,
                         num_key_value_heads=2, head_dim=64, vocab_size=128)
    ids = torch.randint(0, 128, (2, 12), generator=torch.Generator().manual_seed(4)).cuda()
    with torch.no_grad():
        before = model(ids).logits.float()
        pkg.quantize_model_(model, mode)
        after = model(ids).logits.float()
    layer = model.model.layers[0]
    assert isinstance(layer.self_attn.q_proj, pkg.Fp4Linear) and isinstance(layer.mlp, pkg.Fp4GluMLP)
    assert isinstance(layer.input_layernorm, pkg.Fp8RMSNorm) == (mode == "w4a8")
    assert isinstance(model.lm_head, pkg.PackedBf16Linear) and model.dtype == torch.bfloat16
    # Rounding weights to e2m1 moves each by at most a quarter of itself: the logits stay close to the model's.
    assert float((after - before).norm() / before.norm()) < 0.5
    assert bool(torch.isfinite(after).all())
    with pytest.raises(RuntimeError, match="no 4-bit weights"):
        pkg.save_int8_checkpoint(model, "/nonexistent/never-written.safetensors")


def test_quantized_llama_is_refused_whole(pkg):
    """What a mode cannot take is refused before any projection is swapped."""
    from transformers import LlamaConfig, LlamaForCausalLM

    def model(hidden, intermediate, layers=1):
        return LlamaForCausalLM(LlamaConfig(
            hidden_size=hidden, intermediate_size=intermediate, num_hidden_layers=layers, num_attention_heads=2,
            num_key_value_heads=1, vocab_size=64)).to(torch.bfloat16).cuda()

    def kinds(m):
        return [type(x) for x in m.modules()]

    for m, mode, word in ((model(64, 80), "w4a16", "in_features"), (model(48, 64), "w4a8", "in_features"),
                          (pkg.quantize_model_(model(64, 64), "int8"), "w4a8", "already"),
                          (pkg.quantize_model_(model(64, 64), "w8a8"), "w4a16", "already"),
                          (pkg.quantize_model_(model(64, 64), "w4a16"), "int8", "already"),
                          (pkg.quantize_model_(model(64, 64), "w4a8"), "w4a16", "already"),
                          (pkg.quantize_model_(model(64, 64), "w4a8"), "w4a8", "already")):
        before = kinds(m)
        with pytest.raises(RuntimeError, match=word):
            pkg.quantize_model_(m, mode)
        assert kinds(m) == before
    wide = model(64, 64)
    wide.model.layers[0].input_layernorm.weight = torch.nn.Parameter(torch.ones(16416, dtype=torch.bfloat16).cuda())
    with pytest.raises(RuntimeError, match="16384"):
        pkg.quantize_model_(wide, "w4a8")


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 256, 1024), (16, 64, 640), (40, 2048, 512), (100, 128, 4096), (200, 256, 14336), (300, 512, 1024)])
def test_products_replay_from_a_graph_on_another_stream(pkg, rows, m, n, k):
    """Streaming kernel, tiles and tiles with K split (their sums in a workspace), with eager calls in between."""
    code, byte = random_weight(n, k, m)
    w = weight(pkg, code, byte)
    x = activations(m, k, m + 1).cuda()

    def call(x):
        return pkg.ops.w4a8_linear(pkg.ops.quantize_rows_fp8(x), w) if rows else pkg.ops.w4a16_linear(x, w)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call(x)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = call(x)
    for i in range(4):
        fresh = activations(m, k, 100 + i).cuda()
        eager = call(fresh).clone()
        x.copy_(fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


def test_two_graphs_whose_products_split_k(pkg):
    """Each captured call has its own workspace: two graphs replayed on two streams at once do not meet."""
    calls = []
    for i in range(2):
        w = weight(pkg, *random_weight(256, 14336, i))
        x = activations(200, 14336, i).cuda()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            want = pkg.ops.w4a16_linear(x, w)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                got = pkg.ops.w4a16_linear(x, w)
        calls.append((graph, stream, got, want))
    for _ in range(5):
        for graph, stream, _, _ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, got, want in calls:
        assert torch.equal(got, want)
