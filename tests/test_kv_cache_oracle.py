"""The 8-bit cache's restatement (`oracle.kv_cache`) against torch's float8 casts and against formulas, and the
rotary tables against transformers' frequencies; no GPU."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import kv_cache as kv


def test_codes_are_torchs_float8():
    codes = torch.arange(256, dtype=torch.uint8)
    values = codes.view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(values, kv.E4M3)
    x = np.concatenate([np.linspace(-448, 448, 40001), np.random.default_rng(0).standard_normal(40000) * 0.02])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(kv.encode(x.astype(np.float64)), want)
    # Halfway between two codes, and next to it.
    half = (kv.E4M3[:126] + kv.E4M3[1:127]) / 2
    got = kv.encode(half)
    assert (got % 2 == 0).all()
    np.testing.assert_array_equal(kv.encode(half * (1 + 2.0 ** -40)), np.arange(1, 127))
    assert kv.encode(np.array([np.inf, -np.inf, np.nan])).tolist() == [127] * 3


def test_scales_are_the_smallest_that_hold_the_values():
    amax = np.array([0.0, 448.0, 448.0001, 896.0, 1.0, 1.75, 1.7500001, 3.3e38, 1e-38, 2.0 ** -149])
    byte = kv.scale_byte(amax)
    s = 2.0 ** (byte - 127.0)
    assert (amax <= 448 * s).all() and ((amax > 448 * s / 2) | (byte == 1)).all()
    assert byte.tolist()[:4] == [1, 127, 128, 128]


@pytest.mark.parametrize("d", [64, 128])
def test_layout_holds_every_element_once(d):
    slot, dim = np.meshgrid(np.arange(16), np.arange(d), indexing="ij")
    for index in (kv.k_index, kv.v_index):
        assert sorted(index(slot, dim, d).ravel()) == list(range(16 * d))


@pytest.mark.parametrize("d,block_size", [(64, 16), (128, 48)])
def test_unpacking_is_the_librarys(pkg, d, block_size):
    """`unpack_fp8_kv` (torch views) against the element-by-element layout, on random codes."""
    rng = np.random.default_rng(d)
    shape = (3, 2, block_size // 16)
    codes = [rng.integers(0, 256, (*shape, 16 * d), dtype=np.uint8) & 0xfe for _ in range(2)]
    scales = rng.integers(120, 135, (*shape, 2), dtype=np.uint8)
    pool = pkg.ops.fp8_kv_pool(3, block_size, 2, d, "cpu")
    assert pool.block_size == block_size
    for t, a in zip(pool, (*codes, scales)):
        t.view(torch.uint8).copy_(torch.from_numpy(a))
    for got, want in zip(pkg.ops.unpack_fp8_kv(pool), kv.unpack((*codes, scales), block_size)):
        np.testing.assert_array_equal(got.double().numpy(), want)


def _hf_frequencies(kind, rotary, theta, scaling):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    cfg = LlamaConfig(hidden_size=4 * rotary, num_attention_heads=4, head_dim=rotary, rope_theta=theta,
                      max_position_embeddings=8192, rope_scaling=scaling)
    return ROPE_INIT_FUNCTIONS[kind](cfg, torch.device("cpu"))


@pytest.mark.parametrize("scaling", [
    dict(rope_type="linear", factor=4.0),
    dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
         original_max_position_embeddings=8192),
    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=2048),
    dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096, beta_fast=16.0,
         beta_slow=2.0, attention_factor=1.25),
])
@pytest.mark.parametrize("rotary,theta", [(64, 10000.0), (128, 500000.0)])
def test_scaled_tables_are_the_models(pkg, scaling, rotary, theta):
    """cos and sin of a few positions against transformers' frequencies, which are fp32: the angle p f is off
    by at most a few 2^-24 p f from there."""
    freq, gain = _hf_frequencies(scaling["rope_type"], rotary, theta, dict(scaling, rope_theta=theta))
    cos, sin = pkg.ops.rope_table(3000, rotary, theta, scaling)
    assert cos.shape == sin.shape == (3000, rotary // 2) and cos.dtype == torch.float32
    for p in (0, 1, 17, 2999):
        angle = p * freq.double()
        bound = gain * (16 * 2.0 ** -24 * angle + 2.0 ** -22)
        assert ((cos[p].double() - gain * torch.cos(angle)).abs() <= bound).all()
        assert ((sin[p].double() - gain * torch.sin(angle)).abs() <= bound).all()


def test_far_angles_keep_their_precision(pkg):
    """Position 10^6 turns the first pair by 10^6 radians: in fp32 that angle is off by up to 0.03, here by
    nothing but the table's own rounding."""
    cos, sin = pkg.ops.rope_table(1_000_001, 16, 10000.0)
    for i in range(8):
        angle = 1e6 / 10000.0 ** (i / 8)
        assert abs(float(cos[-1, i]) - math.cos(angle)) < 1e-7
        assert abs(float(sin[-1, i]) - math.sin(angle)) < 1e-7


def test_table_refusals(pkg):
    for bad in (dict(rotary=15), dict(rotary=0), dict(positions=0), dict(scaling=dict(rope_type="spiral"))):
        with pytest.raises(RuntimeError):
            pkg.ops.rope_table(**{**dict(positions=4, rotary=16), **bad})
    for bad in ((0, 128), (24, 128), (16, 96)):
        with pytest.raises(RuntimeError):
            pkg.ops.fp8_kv_pool(4, bad[0], 8, bad[1], "cpu")


@pytest.mark.parametrize("scaling,what", [
    (dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=2048, mscale=0.7, mscale_all_dim=1.0), "mscale"),
    (dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=2048, truncate=False), "truncate"),
    (dict(rope_type="yarn", factor=4.0), "needs"), (dict(rope_type="linear"), "needs"),
    (dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192), "needs"),
    (dict(rope_type="linear", factor=2.0, rope_theta=500000.0), "theta"),
    (dict(rope_type="default", rope_theta=500000.0), "theta")])
def test_scalings_that_the_table_would_get_wrong(pkg, scaling, what):
    with pytest.raises(RuntimeError, match=what):
        pkg.ops.rope_table(16, 64, 10000.0, scaling)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_a_complex_product(interleaved):
    """Pairs as complex numbers times e^{i angle}, in fp64; half pairs over whole heads also by transformers."""
    from transformers.models.llama.modeling_llama import apply_rotary_pos_emb

    rng = np.random.default_rng(5)
    x, positions = rng.standard_normal((7, 3, 64)), np.array([0, 1, 5, 30, 2, 9, 31])
    for half in (32, 16, 8):
        angle = np.arange(32)[:, None] / 100.0 ** (np.arange(half) / half)
        got = kv.rotate(x, np.cos(angle), np.sin(angle), positions, interleaved, np.float64)
        pair = x[..., :2 * half]
        z = (pair[..., 0::2] + 1j * pair[..., 1::2] if interleaved else pair[..., :half] + 1j * pair[..., half:])
        z = z * np.exp(1j * angle[positions])[:, None]
        want = x.copy()
        if interleaved:
            want[..., 0:2 * half:2], want[..., 1:2 * half:2] = z.real, z.imag
        else:
            want[..., :half], want[..., half:2 * half] = z.real, z.imag
        np.testing.assert_allclose(got, want, rtol=0, atol=1e-14)
        if half == 32 and not interleaved:
            c, s = (torch.from_numpy(np.tile(f(angle[positions]), 2))[None] for f in (np.cos, np.sin))
            q = torch.from_numpy(x).transpose(0, 1)[None]
            hf = apply_rotary_pos_emb(q, q, c, s)[0][0].transpose(0, 1).numpy()
            np.testing.assert_allclose(got, hf, rtol=0, atol=1e-14)


@pytest.mark.parametrize("pieces", [[70], [1] * 70, [5, 40, 1, 24], [16, 16, 38]])
def test_appended_rows_come_back(pieces):
    """Rows appended in pieces: each value is off by half a step of its code at most, once more where its group's
    scale grew; slots behind the last and other blocks are zeros. A row in another's place is far off."""
    rng = np.random.default_rng(len(pieces))
    k, v = (rng.standard_normal((70, 2, 64)).astype(np.float32) for _ in range(2))
    v[30:40] *= 50.0
    pool = (np.zeros((9, 2, 2, 1024), np.uint8), np.zeros((9, 2, 2, 1024), np.uint8), np.ones((9, 2, 2, 2), np.uint8))
    table, at = np.array([[7, 2, 5, 0]], np.int32), 0
    for n in pieces:
        kv.append(pool, k[at:at + n], v[at:at + n], table, [at], [0], [n], 32)
        at += n
    values = kv.unpack(pool, 32)
    for what, x in enumerate((k, v)):
        got = values[what][table[0]].reshape(128, 2, 64)
        step = 2.0 ** (pool[2][..., what].astype(np.int64) - 127)[table[0]].transpose(0, 2, 1).reshape(8, 2)
        tol = 2.0 ** -4 * np.abs(x) + 2.0 ** -9 * step[np.arange(70) // 16][..., None]
        assert (np.abs(got[:70] - x) <= tol).all()
        assert not got[70:].any() and not (np.abs(got[1:71] - x) <= tol).all()
        assert not values[what][[1, 3, 4, 6, 8]].any()
