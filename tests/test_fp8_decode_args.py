"""The decode runner's 8-bit K/V cache without a GPU: its rotary table, and what it refuses."""

from __future__ import annotations

import pytest
import torch

SMALL = dict(hidden_size=128, intermediate_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=64,
             vocab_size=64)


def _runner(pkg, **overrides):
    from llm_serving_engine_amd.decode_step import DecodeRunner, random_llama

    return DecodeRunner(random_llama(1, seed=3, device=torch.device("cpu"), **{**SMALL, **overrides}), 2, 512)


LLAMA3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
              original_max_position_embeddings=128, rope_theta=500000.0)


@pytest.mark.parametrize("scaling", [None, LLAMA3, dict(rope_type="linear", factor=4.0, rope_theta=500000.0)])
def test_rotary_table_is_the_models(pkg, scaling):
    """Against `ops.rope_table`, whose frequencies are fp64: the model's are fp32 and computed by a power and a few
    products and sums, off by a few steps of 2^-23, so an angle by that times the position; cos and sin are rounded
    once."""
    runner = _runner(pkg, **({} if scaling is None else {"rope_parameters": scaling}))
    got = runner._rope_table()
    want = pkg.ops.rope_table(512, 64, 500000.0, scaling)
    for a, b in zip(got, want):
        assert a.shape == b.shape == (512, 32) and a.dtype is torch.float32
        position = torch.arange(512.0)[:, None]
        assert ((a - b).abs() <= position * 2.0 ** -20 + 2.0 ** -23).all()


def test_refusals(pkg):
    runner = _runner(pkg)
    with pytest.raises(RuntimeError, match="enable_fp8_kv"):
        runner.use_attention("paged-fp8")
    with pytest.raises(ValueError, match="unknown attention"):
        runner.use_attention("fp8")
    with pytest.raises(ValueError, match="needs a GPU"):
        runner.enable_fp8_kv()
    assert runner.attention == "torch" and runner.k_cache[0] is not None and runner.fp8_kv is None


def test_refuses_frequencies_that_change_with_the_length(pkg):
    runner = _runner(pkg, rope_parameters=dict(rope_type="dynamic", factor=2.0, rope_theta=500000.0))
    with pytest.raises(ValueError, match="fixed frequencies"):
        runner._rope_table()
