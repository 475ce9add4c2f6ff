"""`DecodeRunner.enable_fp8_kv` is all or nothing: where it fails, the runner goes on as before."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPE = dict(hidden_size=512, intermediate_size=512, vocab_size=500, num_attention_heads=4, num_key_value_heads=2)


def _runner(dev):
    from llm_serving_engine_amd.decode_step import DecodeRunner, random_llama

    return DecodeRunner(random_llama(3, seed=5, device=dev, **SHAPE), 2, 100)


def _tokens(shape, seed, dev):
    return torch.randint(0, 500, shape, generator=torch.Generator().manual_seed(seed)).to(dev)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("what,layer", [("fp8_kv_pool", 0), ("fp8_kv_pool", 1), ("append_kv_fp8", 0),
                                        ("append_kv_fp8", 2)])
def test_a_failure_leaves_the_runner_as_it_was(pkg, dev, monkeypatch, what, layer, paged):
    runner = _runner(dev)
    if paged:
        runner.enable_paged(block_size=32, seed=3)
        runner.use_attention("paged")
    runner.prefill(_tokens((2, 40), 1, dev))
    tok = _tokens((2,), 2, dev)
    want = runner.step(tok, 40).clone()
    before = {k: v for k, v in vars(runner).items() if k != "_plan"}
    lists = {k: list(v) for k, v in before.items() if isinstance(v, list)}
    real, calls = getattr(pkg.ops, what), []

    def failing(*args, **kw):
        calls.append(None)
        if len(calls) > layer:
            raise torch.OutOfMemoryError("none left")
        return real(*args, **kw)

    with monkeypatch.context() as m:
        m.setattr(pkg.ops, what, failing)
        with pytest.raises(torch.OutOfMemoryError):
            runner.enable_fp8_kv()
    assert len(calls) == layer + 1
    after = vars(runner)
    for name, value in before.items():
        assert after[name] is value, name
    for name, items in lists.items():
        assert all(a is b for a, b in zip(after[name], items)), name
    assert not hasattr(runner, "rope") and runner.fp8_kv is None
    assert torch.equal(runner.step(tok, 40), want)
    # And where it succeeds, nothing of the bf16 caches is left.
    runner.enable_fp8_kv()
    assert runner.attention == "paged-fp8" and runner.k_pool is None and runner.v_pool is None
    assert all(c is None for c in (*runner.k_cache, *runner.v_cache))
    got = runner.step(tok, 40)
    assert (got.float() - want.float()).norm() / want.float().norm() < 0.125
