"""Plain numpy restatement of the 8-bit paged K/V cache: float8 e4m3 codes, power-of-two scales of 16
positions, the pool's byte layout element by element, and the append with its rotation. Slow on purpose;
tests compare the kernels with it. Products and sums of the rotation are rounded in fp32 one by one, so
codes and scales have one right value."""

from __future__ import annotations

import numpy as np

GROUP = 16
NAN_SCALE = 255


def _decode_table() -> np.ndarray:
    """The value of every e4m3 code: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7f and 0xff NaN."""
    out = np.empty(256, np.float64)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        value = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        if c & 127 == 127:
            value = np.nan
        out[c] = -value if c & 128 else value
    return out


E4M3 = _decode_table()


def encode(x: np.ndarray) -> np.ndarray:
    """fp64 values within 448 to the nearest code, ties to the even one; not finite: NaN (0x7f)."""
    x = np.asarray(x, np.float64)
    finite = np.isfinite(x)
    a = np.where(finite, np.abs(x), 0.0)
    assert a.max(initial=0.0) <= 448.0
    grid = E4M3[:127]
    hi = np.clip(np.searchsorted(grid, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    down, up = a - grid[lo], grid[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = np.where(a == grid[hi], hi, code)
    code = code | np.where(np.signbit(x), 128, 0)
    return np.where(finite, code, 127).astype(np.uint8)


def scale_byte(amax: np.ndarray) -> np.ndarray:
    """e8m0 byte of the smallest power of two s >= 2^-126 with amax <= 448 s."""
    amax = np.asarray(amax, np.float64)
    out = np.ones(amax.shape, np.int64)
    for byte in range(1, 254):
        out[amax > 448.0 * 2.0 ** (byte - 127)] = byte + 1
    return out


def keep_finite(codes: np.ndarray, byte: int) -> np.ndarray:
    """Codes of finite values at the scale 2^(byte - 127): those that stand for 2^128 or more, infinity in fp32 and
    bf16, become the largest that does not. NaN stays."""
    below = E4M3[:127] * 2.0 ** (byte - 127) < 2.0 ** 128
    most = np.flatnonzero(below)[-1]
    size = codes & 127
    return np.where((size != 127) & (size > most), codes & 128 | most, codes).astype(np.uint8)


def k_index(slot, d, dim: int):
    return ((slot // 4 * (dim // 64) + d // 64) * 4 + slot % 4) * 64 + d % 64


def v_index(slot, d, dim: int):
    return GROUP * d + slot


def rotate(x: np.ndarray, cos: np.ndarray, sin: np.ndarray, positions, interleaved: bool,
           dtype=np.float32) -> np.ndarray:
    """x (tokens, heads, D) rotated to positions by tables (rows, half), every operation rounded to dtype."""
    out = x.astype(dtype).copy()
    half = cos.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = (t[positions, i].astype(dtype)[:, None] for t in (cos, sin))
        xa, xb = x[..., a].astype(dtype), x[..., b].astype(dtype)
        out[..., a] = xa * c - xb * s
        out[..., b] = xb * c + xa * s
    return out


def append(pool, k, v, table, query_offset, q_start, q_len, block_size: int) -> None:
    """Writes fp32 rows k (already rotated) and v (tokens, H_KV, D) into pool = (k codes, v codes, scales), uint8
    arrays in the pool's layout, in place. Positions past the table, blocks outside the pool and rows outside k and v
    are dropped."""
    kc, vc, scales = pool
    d, n_kv, tokens = k.shape[2], k.shape[1], k.shape[0]
    per = block_size // GROUP
    dims = np.arange(d)
    for e in range(len(q_len)):
        n, off = int(q_len[e]), int(query_offset[e])
        if n <= 0 or off < 0:
            continue
        for g in range(off // GROUP, (off + n - 1) // GROUP + 1):
            if g // per >= table.shape[1]:
                continue
            block, sub = int(table[e, g // per]), g % per
            if not 0 <= block < kc.shape[0]:
                continue
            slots = [s for s in range(GROUP) if off <= g * GROUP + s < off + n]
            rows = [int(q_start[e]) + g * GROUP + s - off for s in slots]
            if not any(0 <= r < tokens for r in rows):
                continue
            lo = slots[0]
            for what, (codes, rows_of, index) in enumerate(((kc, k, k_index), (vc, v, v_index))):
                for h in range(n_kv):
                    new = {s: rows_of[r, h] for s, r in zip(slots, rows) if 0 <= r < tokens}
                    finite = [np.abs(x[np.isfinite(x)]).max(initial=0.0) for x in new.values()]
                    byte = int(scale_byte(np.array(max(finite, default=0.0))))
                    old = int(scales[block, h, sub, what])
                    if lo:
                        byte = max(byte, 0 if old == NAN_SCALE else old)
                    image = np.zeros(GROUP * d, np.uint8)
                    for s in range(lo):
                        was = codes[block, h, sub, index(s, dims, d)]
                        if byte != old:
                            ratio = np.nan if old == NAN_SCALE else 2.0 ** (old - byte)
                            was = encode(E4M3[was] * ratio)
                        image[index(s, dims, d)] = was
                    for s, x in new.items():
                        image[index(s, dims, d)] = keep_finite(encode(x.astype(np.float64) * 2.0 ** (127 - byte)), byte)
                    codes[block, h, sub] = image
                    scales[block, h, sub, what] = byte


def unpack(pool, block_size: int):
    """(k, v) of a pool as fp64 (blocks, block_size, H_KV, D)."""
    kc, vc, scales = pool
    blocks, n_kv, per, size = kc.shape
    d = size // GROUP
    slot, dim = np.meshgrid(np.arange(GROUP), np.arange(d), indexing="ij")
    got = []
    for what, (codes, index) in enumerate(((kc, k_index), (vc, v_index))):
        factor = np.where(scales[..., what] == NAN_SCALE, np.nan, 2.0 ** (scales[..., what].astype(np.int64) - 127))
        x = E4M3[codes[..., index(slot, dim, d)]] * factor[..., None, None]
        got.append(x.transpose(0, 2, 3, 1, 4).reshape(blocks, per * GROUP, n_kv, d))
    return got
