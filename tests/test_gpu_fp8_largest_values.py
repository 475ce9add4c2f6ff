"""The largest finite values in the 8-bit K/V cache: what a scale and a code stand for is finite, and within half a
step of the value."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from fp8_kv_helpers import bf16_rows, i32, pool_to_dev, pool_to_host, random_pool, same_pool, to_dev
from oracle import kv_cache as kv

pytestmark = pytest.mark.gpu

TOP = 2.0 ** 120  # the largest scale that finite values take


def _rows(rng, d):
    """16 tokens of 2 heads with every multiple of 2^120 from 224 to 255 (all that bf16 has there) and both signs,
    the others far below."""
    x = bf16_rows(rng, 16, 2, d)
    top = np.arange(224, 256) * TOP
    x[3, 0, :32], x[5, 1, 8:40], x[15, 1, d - 32:] = top, -top, top[::-1]
    return x.astype(np.float32)


def _append(pkg, dev, pool, k, v, offset, cos=None, sin=None):
    one = i32([len(k)], dev)
    pkg.ops.append_kv_fp8(None, to_dev(k, dev), to_dev(v, dev), cos, sin, pool, i32([[1, 0]], dev),
                          i32([offset], dev), i32([0], dev), one, len(k))
    torch.cuda.synchronize()


@pytest.mark.parametrize("d", [64, 128])
def test_finite_values_stay_finite(pkg, dev, d):
    """Codes round to 256 from 248 up, which 2^120 makes infinite: those are held as 240, at most 15 / 255 < 2^-4
    of the value away."""
    rng = np.random.default_rng(d)
    k, v = _rows(rng, d), _rows(rng, d)
    host = random_pool(rng, 2, 16, 2, d)
    pool = pool_to_dev(pkg, host, dev)
    _append(pkg, dev, pool, k, v, 0)
    kv.append(host, k, v, np.array([[1, 0]]), [0], [0], [16], 16)
    same_pool(pool_to_host(pool), host)
    for got, x in zip(pkg.ops.unpack_fp8_kv(pool), (k, v)):
        got = got[1].double().cpu().numpy()
        assert np.isfinite(got).all()
        loud = np.abs(x) >= 2.0 ** -6 * TOP
        assert loud.sum() == 96
        assert (np.abs(got - x)[loud] <= 2.0 ** -4 * np.abs(x)[loud]).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotated_rows_above_bf16s_largest(pkg, dev, interleaved):
    """A rotation in fp32 gives k values above bf16's largest (255.99 x 2^120, say)."""
    rng = np.random.default_rng(3)
    cos = torch.full((16, 32), 0.8, device=dev)
    sin = torch.full((16, 32), -0.6, device=dev)
    k, v = bf16_rows(rng, 16, 2, 64), bf16_rows(rng, 16, 2, 64)
    a, b = (slice(0, 64, 2), slice(1, 64, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    k[2, 0, a], k[2, 0, b] = 205 * TOP, 153 * TOP  # 0.8 x 205 + 0.6 x 153 = 255.8
    host = random_pool(rng, 2, 16, 2, 64)
    pool = pool_to_dev(pkg, host, dev)
    one = i32([16], dev)
    pkg.ops.append_kv_fp8(None, to_dev(k, dev), to_dev(v, dev), cos, sin, pool, i32([[1, 0]], dev), i32([0], dev),
                          i32([0], dev), one, 16, interleaved=interleaved)
    torch.cuda.synchronize()
    turned = kv.rotate(k, cos.cpu().numpy(), sin.cpu().numpy(), np.arange(16), interleaved)
    assert np.abs(turned).max() > 255.5 * TOP and np.isfinite(turned).all()
    kv.append(host, turned, v, np.array([[1, 0]]), [0], [0], [16], 16)
    same_pool(pool_to_host(pool), host)
    assert torch.isfinite(pkg.ops.unpack_fp8_kv(pool)[0][1].float()).all()


def test_under_a_larger_former_scale(pkg, dev):
    """A half-filled group whose former scale is above 2^120 (another writer's): the rows appended to it are
    finite, the largest code below 2^128 being 1.875 x 2^(128 - 1) at 2^127 and so on."""
    rng = np.random.default_rng(4)
    for byte in (247, 248, 251, 254):
        host = random_pool(rng, 2, 16, 2, 64)
        for codes in host[:2]:
            codes[1] = 0
        host[2][1] = byte
        pool = pool_to_dev(pkg, host, dev)
        k, v = _rows(rng, 64)[:8], _rows(rng, 64)[8:]
        _append(pkg, dev, pool, k, v, 4)
        kv.append(host, k, v, np.array([[1, 0]]), [4], [0], [8], 16)
        same_pool(pool_to_host(pool), host)
        for got, x in zip(pkg.ops.unpack_fp8_kv(pool), (k, v)):
            got = got[1, 4:12].double().cpu().numpy()
            assert np.isfinite(got).all()
            loud = np.abs(x) >= 224 * TOP
            assert (np.abs(got - x)[loud] <= 2.0 ** -4 * np.abs(x)[loud]).all()


def test_infinities_and_nan_are_nan_beside_them(pkg, dev):
    """The largest values' bound is no bound on what is not finite."""
    rng = np.random.default_rng(5)
    k, v = _rows(rng, 64), _rows(rng, 64)
    k[3, 0, 40], k[4, 1, 7], v[5, 1, 0], v[6, 0, 1] = np.inf, np.nan, -np.inf, np.nan
    host = random_pool(rng, 2, 16, 2, 64)
    pool = pool_to_dev(pkg, host, dev)
    _append(pkg, dev, pool, k, v, 0)
    kv.append(host, k, v, np.array([[1, 0]]), [0], [0], [16], 16)
    same_pool(pool_to_host(pool), host)
    for got, x in zip(pkg.ops.unpack_fp8_kv(pool), (k, v)):
        got = got[1].double().cpu().numpy()
        np.testing.assert_array_equal(np.isnan(got), ~np.isfinite(x))
        assert np.isfinite(got[np.isfinite(x)]).all()


@pytest.mark.parametrize("byte", [0, 1, 2, 3, 4, 127, 246])
def test_what_a_code_stands_for(pkg, dev, byte):
    """Attention over one key gives its V row: code x scale exactly from a scale of 2^-124 on, below that rounded to
    bf16's subnormals, whose step is 2^-133; the same as unpacking."""
    pool = pkg.ops.fp8_kv_pool(1, 16, 2, 128, dev)
    codes = torch.arange(256, dtype=torch.uint8, device=dev).view(2, 128)
    codes = torch.where(codes & 127 == 127, torch.zeros_like(codes), codes)
    pool.v.view(torch.uint8).view(1, 2, 1, 128, 16)[0, :, 0, :, 0] = codes
    pool.scales.view(torch.uint8).fill_(byte)
    q = torch.zeros(2, 1, 128, dtype=torch.bfloat16, device=dev)
    one, zero = i32([1], dev), i32([0], dev)
    o = pkg.ops.paged_attention_fp8(q, pool, i32([[0]], dev), one, zero, zero, one, 1)
    exact = codes.view(torch.float8_e4m3fn).double() * 2.0 ** (byte - 127)
    assert ((o[:, 0].double() - exact).abs() <= (0.0 if byte >= 3 else 2.0 ** -134)).all()
    assert torch.equal(o[:, 0], pkg.ops.unpack_fp8_kv(pool)[1][0, 0])
