"""The decode runner over the 8-bit K/V cache: its appends and its attention against the fp64 oracles on what each
layer saw, prompts, decode steps and chunks behind them; and the whole against the bf16 cache."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fp8_kv_helpers import attention_golden
from helpers import bf16_bits
from oracle import kv_cache as kv
from oracle import numerics as ora

pytestmark = pytest.mark.gpu

SHAPE = dict(hidden_size=1024, intermediate_size=2048, vocab_size=1000)


def _runner(dev, batch=3, capacity=300, **overrides):
    from llm_serving_engine_amd.decode_step import DecodeRunner, random_llama

    return DecodeRunner(random_llama(2, seed=21, device=dev, **{**SHAPE, **overrides}), batch, capacity)


def _tokens(shape, seed, dev):
    return torch.randint(0, SHAPE["vocab_size"], shape, generator=torch.Generator().manual_seed(seed)).to(dev)


def _host(pool):
    torch.cuda.synchronize()
    return tuple(t.view(torch.uint8).cpu().numpy() for t in pool)


@pytest.mark.parametrize("h,h_kv,d,backend", [(8, 2, 128, "bf16"), (16, 8, 64, "int8")])
def test_every_layer_appends_and_attends(pkg, dev, monkeypatch, h, h_kv, d, backend):
    """Each layer's cache codes equal the oracle's append of the projections, bit for bit, and each layer's
    attention output is within its tolerance of fp64 over them."""
    runner = _runner(dev, num_attention_heads=h, num_key_value_heads=h_kv, head_dim=d)
    if backend == "int8":
        runner.quantize("int8")
    runner.use(backend)
    runner.enable_fp8_kv(block_size=32)
    calls = []
    append, attend = pkg.ops.append_kv_fp8, pkg.ops.paged_attention_fp8

    def seen_append(q, k, v, cos, sin, pool, *plan):
        before = _host(pool)
        out = append(q, k, v, cos, sin, pool, *plan)
        calls.append((before, _host(pool), [bf16_bits(t) for t in (q, k, v)], bf16_bits(out)))
        return out

    def seen_attend(q, pool, *plan):
        o = attend(q, pool, *plan)
        calls[-1] += (bf16_bits(q), bf16_bits(o), [t.cpu().numpy() for t in plan[:-1]])
        return o

    monkeypatch.setattr(pkg.ops, "append_kv_fp8", seen_append)
    monkeypatch.setattr(pkg.ops, "paged_attention_fp8", seen_attend)
    cos, sin = (t.cpu().numpy() for t in runner.rope)
    for start, ntok, rows in [(0, 150, slice(0, 2)), (0, 150, slice(2, 3)), (150, 1, None), (151, 1, None),
                              (152, 40, slice(1, 3))]:
        calls.clear()
        runner.forward(_tokens((3 if rows is None else rows.stop - rows.start, ntok), start, dev), start, rows)
        assert len(calls) == 2
        for before, after, (q, k, v), q_out, q_in, o, (table, ctx, qo, qs, ql) in calls:
            want = tuple(a.copy() for a in before)
            q, k, v = (ora.bf16_bits_to_f32(a) for a in (q, k, v))
            pos = np.concatenate([np.arange(a, a + n) for a, n in zip(qo, ql)])
            q, k = (kv.rotate(x, cos, sin, pos, False) for x in (q, k))
            kv.append(want, k, v, table, qo, qs, ql, 32)
            for a, b in zip(after, want):
                np.testing.assert_array_equal(a, b)
            np.testing.assert_array_equal(q_out, ora.f32_to_bf16_bits(q))
            np.testing.assert_array_equal(q_in, q_out.transpose(1, 0, 2))
            case = dict(q=q_in, pool=after, bs=32, table=table, ctx=ctx, qo=qo, qs=qs, ql=ql)
            golden, covered, vmax = attention_golden(case)
            assert covered.all()
            ok, msg = ora.attention_within_tolerance(o, golden, vmax, covered)
            assert ok, msg


@pytest.mark.parametrize("when", ["before", "after"])
def test_logits_track_the_bf16_cache(pkg, dev, when):
    """Prompts and three decode steps, the cache made 8-bit before or after the prompts. A value of k or v is off by
    2^-4 of it at most and a score by less than that of itself, so an attention output by less than an eighth of the
    values it averages; it is one term of the residual sum."""
    prompt = _tokens((3, 100), 1, dev)
    ref, runner = (_runner(dev) for _ in range(2))
    ref.prefill(prompt)
    if when == "before":
        runner.enable_fp8_kv()
    runner.prefill(prompt)
    if when == "after":
        runner.enable_fp8_kv()
    assert runner.attention == "paged-fp8" and runner.k_cache[0] is None
    tok = _tokens((3,), 2, dev)
    for t in range(3):
        want, got = (r.step(tok, 100 + t).float() for r in (ref, runner))
        assert (got - want).norm() / want.norm() < 0.125
        tok = want.argmax(-1)


def test_sequences_by_index(pkg, dev):
    """Sequences given by index, in another order than their slice: the same hidden states."""
    runner = _runner(dev)
    runner.enable_fp8_kv()
    runner.prefill(_tokens((3, 40), 6, dev))
    tok = _tokens((2, 3), 7, dev)
    want = runner.forward(tok, 40, slice(1, 3)).reshape(2, 3, -1)
    for rows in ([2, 1], torch.tensor([2, 1], device=dev)):
        got = runner.forward(tok.flip(0), 40, rows).reshape(2, 3, -1)
        assert torch.equal(got.flip(0), want)


def test_a_step_replays_from_a_graph(pkg, dev):
    """One decode step, captured; replays with eager steps between are the eager step's bits."""
    runner = _runner(dev)
    runner.enable_fp8_kv()
    runner.prefill(_tokens((3, 70), 3, dev))
    tok = _tokens((3,), 4, dev)
    eager = runner.step(tok, 70).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        runner.step(tok, 70)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = runner.step(tok, 70)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(runner.step(tok, 70), eager)


def test_refusals(pkg, dev):
    runner = _runner(dev, capacity=40)
    with pytest.raises(ValueError, match="block_size"):
        runner.enable_fp8_kv(block_size=24)
    assert runner.k_cache[0] is not None
    runner.enable_fp8_kv()
    for kind in ("torch", "paged"):
        with pytest.raises(RuntimeError, match="8-bit"):
            runner.use_attention(kind)
    for call in (runner.enable_paged, runner.enable_fp8_kv):
        with pytest.raises(RuntimeError, match="8-bit"):
            call()
    with pytest.raises(ValueError, match="capacity"):
        runner.forward(_tokens((3, 2), 5, dev), 39)
    full = _runner(dev)
    full.model.float()
    with pytest.raises(ValueError, match="bf16 model"):
        full.enable_fp8_kv()
    wide = _runner(dev, num_attention_heads=32, num_key_value_heads=1, head_dim=64)
    with pytest.raises(ValueError, match="query heads"):
        wide.enable_fp8_kv()
