"""Tensor-level ops over the C ABI. Each validates dtypes, devices and layouts in Python,
allocates its outputs with `torch.empty` (so CUDA-graph memory pools own them), and enqueues
the HIP kernel on the current stream without synchronising, which keeps every op capturable
into a graph.

Weights are held in the packed tile layout the kernels stream (`pack_weight`): a (N, K) int8
matrix becomes a (ceil(N/16), ceil(K/64), 1024) int8 tensor whose 1 KB tiles are 16 rows x 64
K-bytes each, in matrix-core operand order. The MLP's gate and up weights share one tensor in the
gate/up layout (`pack_glu`): row tile 2t holds gate rows 16t..16t+15, row tile 2t+1 the same up
rows, so one kernel computes both and applies SiLU-mul before anything leaves registers.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib

__all__ = [
    "Fp4Weight",
    "Fp8KV",
    "Fp8Rows",
    "add_rmsnorm",
    "add_rmsnorm_fp8",
    "append_kv_fp8",
    "bf16_decode_linear",
    "dequantize_fp4",
    "dequantize_rows_fp8",
    "fp8_kv_pool",
    "pack_bf16_weight",
    "packed_bf16_shape",
    "unpack_bf16_weight",
    "paged_attention_forward",
    "paged_attention_fp8",
    "pack_fp4",
    "pack_glu",
    "pack_weight",
    "packed_glu_shape",
    "packed_shape",
    "quantize_act_per_token",
    "quantize_rows_fp8",
    "quantize_weight_fp4",
    "quantize_weight_per_channel",
    "rmsnorm_quantize",
    "rope",
    "rope_kv",
    "rope_table",
    "unpack_fp4",
    "unpack_fp8_kv",
    "unpack_glu",
    "unpack_weight",
    "w8a8_gemm",
    "w8a8_glu",
    "w8a8_glu_quantized",
    "w8a8_linear",
    "w4a16_glu",
    "w4a16_linear",
    "w4a8_glu",
    "w4a8_linear",
    "w8a16_glu",
    "w8a16_linear",
    "w8a16_linear_noalloc",
    "workspace",
]


# A decode call's kernel runs 5 to 10 us, so the checks before it are written for their cost on the
# host: plain conditions with the message built only to raise it, device indices and raw stream
# handles instead of device and stream objects, and no view of the input or the output where their
# memory already has the rows the kernel takes. An eager `Int8Linear` call of one row went from 18.2
# to about 11 us a call.


def _stream(device: torch.device | int) -> int:
    if not isinstance(device, int):
        device = device.index if device.index is not None else torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(device)


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _on_gpu(first: torch.Tensor, *others: torch.Tensor) -> int:
    """The index of the GPU all of the tensors are on."""
    if not first.is_cuda:
        raise RuntimeError(f"int8 kernels need a CUDA (HIP) device, got {first.device}")
    index = first.get_device()
    for t in others:
        if not t.is_cuda or t.get_device() != index:
            raise RuntimeError(f"tensors on different devices: {first.device} and {t.device}")
    return index


def _rows(x: torch.Tensor, k: int) -> torch.Tensor:
    """(..., K) → a 2-D (rows, K) view whose last dim is contiguous."""
    _require(x.shape[-1] == k, f"expected last dim {k}, got {tuple(x.shape)}")
    x2 = x.reshape(-1, k)
    strided_rows = x2.shape[0] > 1 and (x2.stride(0) < k or x2.stride(0) % 8)
    if x2.stride(-1) != 1 or strided_rows or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    return x2


def _row_args(x: torch.Tensor, k: int) -> tuple[torch.Tensor, int, int, int]:
    """(owner, address, row stride, rows) of x (..., K) as `_rows` gives them; `owner` is to be
    kept until the kernel is enqueued."""
    if k and x.is_contiguous() and x.shape[-1] == k:
        at = x.data_ptr()
        if at % 16 == 0:
            return x, at, k, x.numel() // k
    x2 = _rows(x, k)
    m = x2.shape[0]
    return x2, x2.data_ptr(), x2.stride(0) if m > 1 else k, m


# ---- packed weights --------------------------------------------------------------------------


def packed_shape(n: int, k: int) -> tuple[int, int, int]:
    return ((n + 15) // 16, (k + 63) // 64, 1024)


def pack_weight(q: torch.Tensor) -> torch.Tensor:
    """Row-major (N, K) int8 → packed (ceil(N/16), ceil(K/64), 1024) int8, on the GPU."""
    _require(q.dim() == 2 and q.dtype == torch.int8, "q must be a 2-D int8 tensor")
    dev = _on_gpu(q)
    n, k = q.shape
    q = q.contiguous()
    qp = torch.empty(packed_shape(n, k), dtype=torch.int8, device=dev)
    _lib.check(_lib.library().lse_pack_weight(q.data_ptr(), n, k, qp.data_ptr(), _stream(dev)),
               "lse_pack_weight")
    return qp


def unpack_weight(qp: torch.Tensor, n: int, k: int) -> torch.Tensor:
    """Inverse of `pack_weight` (a pure permutation, done with torch views): (N, K) int8."""
    rb, steps, _ = qp.shape
    t = qp.reshape(rb, steps, 4, 16, 16)  # [rb][step][g = lane // 16][row = lane % 16][16 bytes]
    t = t.permute(0, 3, 1, 2, 4).reshape(rb * 16, steps * 64)
    return t[:n, :k].contiguous()


def packed_glu_shape(i: int, k: int) -> tuple[int, int, int]:
    return (2 * ((i + 15) // 16), (k + 63) // 64, 1024)


def pack_glu(q: torch.Tensor) -> torch.Tensor:
    """Stacked row-major (2I, K) int8 [gate; up] → the gate/up layout, (2 ceil(I/16), ceil(K/64),
    1024) int8, on the GPU."""
    _require(q.dim() == 2 and q.dtype == torch.int8 and q.shape[0] % 2 == 0,
             "q must be a 2-D int8 tensor of 2I stacked gate and up rows")
    dev = _on_gpu(q)
    i, k = q.shape[0] // 2, q.shape[1]
    q = q.contiguous()
    qp = torch.empty(packed_glu_shape(i, k), dtype=torch.int8, device=dev)
    _lib.check(_lib.library().lse_pack_glu(q.data_ptr(), i, k, qp.data_ptr(), _stream(dev)),
               "lse_pack_glu")
    return qp


def unpack_glu(qp: torch.Tensor, i: int, k: int) -> torch.Tensor:
    """Inverse of `pack_glu`: the stacked (2I, K) int8 [gate; up]."""
    rows = unpack_weight(qp, qp.shape[0] * 16, k)  # packed rows, tile pairs (gate, up)
    pairs = rows.reshape(-1, 2, 16, k)
    gate = pairs[:, 0].reshape(-1, k)[:i]
    up = pairs[:, 1].reshape(-1, k)[:i]
    return torch.cat([gate, up]).contiguous()


def workspace(mode: int, m: int, n: int, k: int,
              dev: torch.device | int) -> torch.Tensor | None:
    """The workspace one GEMM call needs (deep decode shapes and 65..256 tokens over a narrow
    weight add partial sums of K ranges in a second pass), or None. Allocated with torch.empty,
    so graph-pool owned under capture; the caller keeps it alive until the call is enqueued."""
    nbytes = _lib.library().lse_workspace_bytes(mode, m, n, k)
    if nbytes < 0:
        raise RuntimeError(f"lse_workspace_bytes rejected (M, N, K) = ({m}, {n}, {k})")
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _ws_args(ws: torch.Tensor | None) -> tuple[int | None, int]:
    return (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)


def _check_packed(qp: torch.Tensor, n: int, k: int, glu: bool = False) -> None:
    if qp.dtype is not torch.int8 or not qp.is_contiguous():
        raise RuntimeError("packed weight must be contiguous int8")
    want = packed_glu_shape(n, k) if glu else packed_shape(n, k)
    if qp.shape != want:
        what = "(I, K)" if glu else "(N, K)"
        raise RuntimeError(f"packed weight has shape {tuple(qp.shape)}, {what} = ({n}, {k}) needs "
                           f"{want}")


def _check_bf16(x: torch.Tensor, what: str) -> None:
    if x.dtype is not torch.bfloat16:
        raise RuntimeError(f"{what} expects bf16 activations, got {x.dtype}")


def _channel_scales(scales: torch.Tensor) -> int:
    if scales.dtype is not torch.float32 or scales.dim() != 1:
        raise RuntimeError("scales must be fp32 (N,)")
    return scales.shape[0]


def _glu_scales(scales: torch.Tensor) -> int:
    if scales.dtype is not torch.float32 or scales.dim() != 1 or scales.shape[0] % 2:
        raise RuntimeError("gate/up scales must be fp32 (2I,) [gate; up]")
    return scales.shape[0] // 2


# ---- ops -------------------------------------------------------------------------------------


def quantize_weight_per_channel(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """W (N, K) → (q (N, K) int8 row-major, s (N,) fp32), s = amax/127 per row, q = clamp(rne(W/s)).

    Runs on the GPU at load time. W is read as fp32 (bf16/fp16 weights widen exactly).
    """
    _require(w.dim() == 2, f"weight must be 2-D, got {tuple(w.shape)}")
    dev = _on_gpu(w)
    n, k = w.shape
    w32 = w.to(torch.float32).contiguous()
    q = torch.empty((n, k), dtype=torch.int8, device=dev)
    s = torch.empty((n,), dtype=torch.float32, device=dev)
    lib = _lib.library()
    _lib.check(
        lib.lse_quantize_weight_per_channel(
            w32.data_ptr(), k, q.data_ptr(), s.data_ptr(), n, k, _stream(dev)
        ),
        "lse_quantize_weight_per_channel",
    )
    return q, s


def w8a16_linear(
    x: torch.Tensor,
    qp: torch.Tensor,
    scales: torch.Tensor,
    algo: int = _lib.ALGO_AUTO,
) -> torch.Tensor:
    """y = bf16(s[n] * sum_k x[..., k] q[n, k]) for x (..., K) bf16 → y (..., N) bf16, with the
    weight q given packed (`pack_weight`)."""
    dev = _on_gpu(x, qp, scales)
    _check_bf16(x, "W8A16")
    n, lead = _channel_scales(scales), x.shape
    k = lead[-1]
    _check_packed(qp, n, k)
    owner, at, ldx, m = _row_args(x, k)
    y = torch.empty((*lead[:-1], n), dtype=torch.bfloat16, device=dev)
    ws = workspace(_lib.MODE_W8A16, m, n, k, dev)
    _lib.check(
        _lib.library().lse_w8a16_gemm_algo(
            at, ldx, qp.data_ptr(), scales.data_ptr(), y.data_ptr(), n, m, n, k, algo,
            *_ws_args(ws), _stream(dev),
        ),
        "lse_w8a16_gemm",
    )
    return y


def w8a16_linear_noalloc(x: torch.Tensor, qp: torch.Tensor, scales: torch.Tensor,
                         out: torch.Tensor) -> torch.Tensor:
    """`w8a16_linear` into a caller-given `out` (M, N) bf16 through `lse_w8a16_gemm_noalloc`:
    nothing is allocated (the decode kernel's split-K partial sums live in the library's static
    per-device scratch). x must already be (M, K) with a contiguous last dim."""
    dev = _on_gpu(x, qp, scales, out)
    _require(x.dtype == torch.bfloat16 and out.dtype == torch.bfloat16, "bf16 x and out expected")
    _require(scales.dtype == torch.float32 and scales.dim() == 1, "scales must be fp32 (N,)")
    _require(x.dim() == 2 and x.stride(-1) == 1, "x must be (M, K) with a contiguous last dim")
    n, (m, k) = scales.shape[0], x.shape
    _check_packed(qp, n, k)
    _require(out.dim() == 2 and tuple(out.shape) == (m, n) and out.stride(-1) == 1,
             f"out must be ({m}, {n}) with a contiguous last dim")
    _lib.check(
        _lib.library().lse_w8a16_gemm_noalloc(
            x.data_ptr(), x.stride(0) if m > 1 else k, qp.data_ptr(), scales.data_ptr(),
            out.data_ptr(), out.stride(0) if m > 1 else n, m, n, k, _stream(dev)),
        "lse_w8a16_gemm_noalloc",
    )
    return out


def quantize_act_per_token(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (..., K) bf16 → (xq (rows, K) int8, sx (rows,) fp32), per-row symmetric int8."""
    dev = _on_gpu(x)
    _check_bf16(x, "W8A8")
    k = x.shape[-1]
    owner, at, ldx, m = _row_args(x, k)
    xq = torch.empty((m, k), dtype=torch.int8, device=dev)
    sx = torch.empty((m,), dtype=torch.float32, device=dev)
    _lib.check(
        _lib.library().lse_quantize_act_per_token(
            at, ldx, xq.data_ptr(), sx.data_ptr(), m, k, _stream(dev)
        ),
        "lse_quantize_act_per_token",
    )
    return xq, sx


def _quantized_rows(xq: torch.Tensor, sx: torch.Tensor, msg: str) -> tuple[int, int]:
    if xq.dim() != 2 or xq.dtype is not torch.int8 or not xq.is_contiguous():
        raise RuntimeError(msg)
    m, k = xq.shape
    if sx.dtype is not torch.float32 or sx.shape != (m,):
        raise RuntimeError("sx must be fp32 (M,)")
    return m, k


def w8a8_gemm(
    xq: torch.Tensor,
    sx: torch.Tensor,
    qp: torch.Tensor,
    scales: torch.Tensor,
    want_acc: bool = False,
    want_y: bool = True,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """(y (M, N) bf16 or None, acc (M, N) int32 or None) from quantized operands; the weight q
    is given packed."""
    dev = _on_gpu(xq, sx, qp, scales)
    n = _channel_scales(scales)
    m, k = _quantized_rows(xq, sx, "xq must be (M, K) int8")
    _check_packed(qp, n, k)
    y = torch.empty((m, n), dtype=torch.bfloat16, device=dev) if want_y else None
    acc = torch.empty((m, n), dtype=torch.int32, device=dev) if want_acc else None
    ws = workspace(_lib.MODE_W8A8, m, n, k, dev)
    _lib.check(
        _lib.library().lse_w8a8_gemm(
            xq.data_ptr(), sx.data_ptr(), qp.data_ptr(), scales.data_ptr(),
            y.data_ptr() if y is not None else None, n,
            acc.data_ptr() if acc is not None else None, m, n, k, *_ws_args(ws), _stream(dev),
        ),
        "lse_w8a8_gemm",
    )
    return y, acc


# Elements of x (M * K) up to which w8a8_linear takes the one-launch kernel.
ONE_LAUNCH_W8A8_MAX_ELEMS = 14336


def w8a8_linear(x: torch.Tensor, qp: torch.Tensor, scales: torch.Tensor,
                want_acc: bool = False, one_launch: bool | None = None):
    """Dynamic per-token W8A8: quantize x per row, int8 GEMM with exact int32 accumulation,
    y = bf16((acc * sx[m]) * s[n]). x (..., K) bf16 → y (..., N) bf16 (with want_acc, also the
    (M, N) int32 accumulators). Up to ONE_LAUNCH_W8A8_MAX_ELEMS elements of x (1 to 3 rows of
    4096, 1 row of 14336) run as one kernel that quantizes while it stages x (`lse_w8a8_linear`);
    more quantize first, then run the GEMM. Both give the same bits. The one-launch kernel
    quantizes all of x in every workgroup, so its cost grows with M * K: measured on MI355X over
    the Llama-3-8B shapes it is 3-16 % faster up to 14336 elements, and 6 % slower at 2 x 14336
    (down_proj) and up to 6 % at 4 x 4096. `one_launch` True takes the one-launch kernel wherever
    it runs (`lse_w8a8_linear_supported`), False never."""
    n, k = scales.shape[0], x.shape[-1]
    lib = _lib.library()
    m = x.numel() // k if k else 0
    if one_launch is None:
        one_launch = m * k <= ONE_LAUNCH_W8A8_MAX_ELEMS
    if m and one_launch and lib.lse_w8a8_linear_supported(m, k):
        dev = _on_gpu(x, qp, scales)
        _check_bf16(x, "W8A8")
        _channel_scales(scales)
        _check_packed(qp, n, k)
        owner, at, ldx, _ = _row_args(x, k)
        y = torch.empty((m, n), dtype=torch.bfloat16, device=dev)
        acc = torch.empty((m, n), dtype=torch.int32, device=dev) if want_acc else None
        _lib.check(
            lib.lse_w8a8_linear(
                at, ldx, qp.data_ptr(), scales.data_ptr(), y.data_ptr(), n,
                acc.data_ptr() if acc is not None else None, m, n, k, _stream(dev),
            ),
            "lse_w8a8_linear",
        )
    else:
        xq, sx = quantize_act_per_token(x)
        y, acc = w8a8_gemm(xq, sx, qp, scales, want_acc=want_acc)
    y = y.view(*x.shape[:-1], n)
    return (y, acc) if want_acc else y


def w8a16_glu(
    x: torch.Tensor,
    qp: torch.Tensor,
    scales: torch.Tensor,
    algo: int = _lib.ALGO_AUTO,
) -> torch.Tensor:
    """h = bf16(silu(g) * u) for x (..., K) bf16 → h (..., I) bf16, where g and u are the fp32
    W8A16 products of x with the gate and up weights (`pack_glu` layout, scales (2I,) [gate;
    up]); one kernel, one rounding."""
    dev = _on_gpu(x, qp, scales)
    _check_bf16(x, "W8A16")
    i, lead = _glu_scales(scales), x.shape
    k = lead[-1]
    _check_packed(qp, i, k, glu=True)
    owner, at, ldx, m = _row_args(x, k)
    h = torch.empty((*lead[:-1], i), dtype=torch.bfloat16, device=dev)
    _lib.check(
        _lib.library().lse_w8a16_glu(
            at, ldx, qp.data_ptr(), scales.data_ptr(), h.data_ptr(), i, m, i, k, algo, _stream(dev),
        ),
        "lse_w8a16_glu",
    )
    return h


def w8a8_glu(x: torch.Tensor, qp: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Dynamic per-token W8A8 form of `w8a16_glu`: x quantized per row, exact int32 sums,
    g = (acc_g * sx) * s_g, u likewise, h = bf16(silu(g) * u). x (..., K) → h (..., I)."""
    xq, sx = quantize_act_per_token(x)
    h = w8a8_glu_quantized(xq, sx, qp, scales)
    return h.view(*x.shape[:-1], h.shape[-1])


def w8a8_glu_quantized(xq: torch.Tensor, sx: torch.Tensor, qp: torch.Tensor,
                       scales: torch.Tensor) -> torch.Tensor:
    """`w8a8_glu` from already quantized rows: xq (M, K) int8, sx (M,) fp32 → h (M, I) bf16."""
    dev = _on_gpu(xq, sx, qp, scales)
    i = _glu_scales(scales)
    m, k = _quantized_rows(xq, sx, "xq must be contiguous (M, K) int8")
    _check_packed(qp, i, k, glu=True)
    h = torch.empty((m, i), dtype=torch.bfloat16, device=dev)
    _lib.check(
        _lib.library().lse_w8a8_glu(
            xq.data_ptr(), sx.data_ptr(), qp.data_ptr(), scales.data_ptr(), h.data_ptr(), i, m, i,
            k, _stream(dev),
        ),
        "lse_w8a8_glu",
    )
    return h


def paged_attention_forward(
    q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
    block_table: torch.Tensor, context_len: torch.Tensor, query_offset: torch.Tensor,
    q_start: torch.Tensor, q_len: torch.Tensor, block_size: int, max_q_len: int,
) -> torch.Tensor:
    """One launch for a whole batch plan's attention at one layer against a shared paged K/V
    pool, with the reference's signature and meaning (`paged_attention_forward`,
    src/llm_serving_engine/kernels/flash_attention.py:287-332).

    q: (H, total_tokens, D) bf16. k_pool/v_pool: (num_blocks, block_size, H_KV, D) bf16, already
    holding this call's tokens. block_table (entries, max_blocks), context_len, query_offset,
    q_start, q_len (entries,): int32 on the device. max_q_len >= every q_len. Returns o like q.
    Softmax scale 1/sqrt(D). D = 128 and 1 <= H / H_KV <= 16 (24 query heads over 8 K/V
    heads included)."""
    entry = (context_len, query_offset, q_start, q_len)
    dev = _on_gpu(q, k_pool, v_pool, block_table, *entry)
    if q.dim() != 3 or k_pool.dim() != 4 or v_pool.shape != k_pool.shape:
        raise RuntimeError("q must be (H, T, D), k_pool/v_pool (num_blocks, block_size, H_KV, D)")
    bf16 = torch.bfloat16
    if q.dtype is not bf16 or k_pool.dtype is not bf16 or v_pool.dtype is not bf16:
        raise RuntimeError(f"paged attention runs on bf16 q/k/v, got {q.dtype}, {k_pool.dtype}, "
                           f"{v_pool.dtype}")
    names = ("context_len", "query_offset", "q_start", "q_len")
    for name, t in zip(("block_table", *names), (block_table, *entry)):
        if t.dtype is not torch.int32:
            raise RuntimeError(f"{name} must be int32, got {t.dtype}")
    if block_table.dim() != 2 or block_table.stride(1) != 1:
        raise RuntimeError("block_table must be (E, B) with unit column stride")
    entries = block_table.shape[0]
    for name, t in zip(names, entry):
        if t.shape != (entries,) or t.stride(0) != 1:
            raise RuntimeError(f"{name} must be a contiguous ({entries},) tensor")
    h, _tokens, d = q.shape
    _, bs, h_kv, dk = k_pool.shape
    if dk != d or bs != block_size:
        raise RuntimeError("pool shape does not match q / block_size")
    if q.stride(2) != 1 or k_pool.stride(3) != 1 or v_pool.stride() != k_pool.stride():
        raise RuntimeError("head dim must be contiguous and k_pool/v_pool must share strides")
    o = torch.empty_like(q)
    lib = _lib.library()
    nbytes = lib.lse_paged_attention_workspace_bytes(entries, h, h_kv, d, max_q_len,
                                                     block_table.shape[1], block_size)
    if nbytes < 0:
        raise RuntimeError(f"unsupported attention shape: H={h} H_KV={h_kv} D={d}")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _lib.check(
        lib.lse_paged_attention(
            q.data_ptr(), q.stride(0), q.stride(1), k_pool.data_ptr(), v_pool.data_ptr(),
            k_pool.stride(0), k_pool.stride(1), k_pool.stride(2), block_table.data_ptr(),
            block_table.stride(0), context_len.data_ptr(), query_offset.data_ptr(),
            q_start.data_ptr(), q_len.data_ptr(), o.data_ptr(), o.stride(0), o.stride(1),
            entries, h, h_kv, d, block_size, block_table.shape[1], max_q_len, 1.0 / d ** 0.5,
            *_ws_args(ws), _stream(dev),
        ),
        "lse_paged_attention",
    )
    return o


def rmsnorm_quantize(
    x: torch.Tensor, weight: torch.Tensor, eps: float, want_normed: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """LlamaRMSNorm (transformers modeling_llama.py:62-67) and per-token int8 quantization of its
    bf16 output in one kernel: x (..., K) bf16, weight (K,) bf16 → (xq (rows, K) int8, sx (rows,)
    fp32, normed (rows, K) bf16 or None)."""
    dev = _on_gpu(x, weight)
    if x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16:
        raise RuntimeError(
            f"RMSNorm-quantize takes bf16 x and weight, got {x.dtype}, {weight.dtype}")
    k = x.shape[-1]
    if weight.shape != (k,):
        raise RuntimeError(f"weight must be ({k},), got {tuple(weight.shape)}")
    owner, at, ldx, m = _row_args(x, k)
    w = weight.contiguous()
    xq = torch.empty((m, k), dtype=torch.int8, device=dev)
    sx = torch.empty((m,), dtype=torch.float32, device=dev)
    normed = torch.empty((m, k), dtype=torch.bfloat16, device=dev) if want_normed else None
    _lib.check(
        _lib.library().lse_rmsnorm_quantize(
            at, ldx, w.data_ptr(), float(eps),
            xq.data_ptr(), sx.data_ptr(), normed.data_ptr() if normed is not None else None, m,
            k, _stream(dev),
        ),
        "lse_rmsnorm_quantize",
    )
    return xq, sx, normed


def add_rmsnorm(
    x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float,
) -> tuple[torch.Tensor, torch.Tensor]:
    """(s, LlamaRMSNorm(s)) with s = x + residual (x itself when residual is None) in one kernel:
    x and residual (..., K) bf16, weight (K,) bf16, K <= `_lib.NORM_MAX_K`."""
    dev = _on_gpu(x, weight) if residual is None else _on_gpu(x, weight, residual)
    k = x.shape[-1]
    _require(x.dtype == weight.dtype == torch.bfloat16 and weight.shape == (k,),
             f"RMSNorm takes bf16 x and weight ({k},)")
    x2 = _rows(x, k)
    m = x2.shape[0]
    y = torch.empty(x.shape, dtype=torch.bfloat16, device=dev)
    if residual is None:
        r2, s = None, x
    else:
        _require(residual.dtype == torch.bfloat16 and residual.shape == x.shape,
                 "the residual must be bf16 and of x's shape")
        r2, s = _rows(residual, k), torch.empty(x.shape, dtype=torch.bfloat16, device=dev)
    w = weight.contiguous()
    if w.data_ptr() % 16:  # a piece of a flat parameter buffer
        w = w.clone()
    _lib.check(
        _lib.library().lse_add_rmsnorm(
            x2.data_ptr(), x2.stride(0) if m > 1 else k,
            r2.data_ptr() if r2 is not None else None,
            r2.stride(0) if r2 is not None and m > 1 else k, w.data_ptr(), float(eps),
            s.data_ptr() if r2 is not None else None, y.data_ptr(), m, k, _stream(dev)),
        "lse_add_rmsnorm",
    )
    return s, y


def rope_kv(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
    n_heads: int, n_kv: int, sequences: int, start: int,
    cache: tuple[torch.Tensor, torch.Tensor] | None = None,
    pool: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
) -> torch.Tensor:
    """Rotates one layer's new q and k (`apply_rotary_pos_emb`, the same bits) and writes k and v at
    positions [start, start + tokens / sequences) of every sequence, in one kernel.

    q (..., n_heads D), k and v (..., n_kv D): bf16, rows of consecutive sequences' tokens, the last
    dim contiguous. cos, sin (tokens, D) bf16. cache: (k, v) of (sequences, n_kv, capacity, D).
    pool: (k, v, table) of (blocks, block_size, n_kv, D) and int32 (sequences, blocks). Returns the
    rotated q as (tokens, n_heads, D)."""
    dev = _on_gpu(q, k, v, cos, sin)
    d = cos.shape[-1]
    rows = []
    for name, t, width in (("q", q, n_heads * d), ("k", k, n_kv * d), ("v", v, n_kv * d),
                           ("cos", cos, d), ("sin", sin, d)):
        _require(t.dtype == torch.bfloat16, f"{name} must be bf16, got {t.dtype}")
        rows.append(_rows(t, width))
    tokens = rows[0].shape[0]
    _require(all(t.shape[0] == tokens for t in rows) and tokens % max(1, sequences) == 0,
             "q, k, v, cos and sin need one row per token of every sequence")
    ntok = tokens // max(1, sequences)
    if rows[4].stride(0) != rows[3].stride(0):
        rows[3], rows[4] = rows[3].contiguous(), rows[4].contiguous()
    out = torch.empty((tokens, n_heads, d), dtype=torch.bfloat16, device=dev)
    cache_args, pool_args = [None, None, 0, 0, 0], [None, None, 0, 0, 0, None, 0, 1]
    if cache is not None:
        kc, vc = cache
        _on_gpu(q, kc, vc)
        _require(kc.dtype == vc.dtype == torch.bfloat16 and kc.shape == vc.shape
                 and kc.stride() == vc.stride() and kc.stride(3) == 1
                 and kc.shape[:2] == (sequences, n_kv) and kc.shape[3] == d
                 and kc.shape[2] >= start + ntok,
                 f"cache must be two bf16 ({sequences}, {n_kv}, >= {start + ntok}, {d}) tensors")
        cache_args = [kc.data_ptr(), vc.data_ptr(), *kc.stride()[:3]]
    if pool is not None:
        kp, vp, table = pool
        _on_gpu(q, kp, vp, table)
        _require(kp.dtype == vp.dtype == torch.bfloat16 and kp.shape == vp.shape
                 and kp.stride() == vp.stride() and kp.stride(3) == 1
                 and kp.shape[2:] == (n_kv, d), f"pool must be two bf16 (*, *, {n_kv}, {d}) tensors")
        _require(table.dtype == torch.int32 and table.dim() == 2 and table.stride(1) == 1
                 and table.shape[0] == sequences
                 and table.shape[1] * kp.shape[1] >= start + ntok,
                 f"table must be int32, {sequences} rows covering {start + ntok} positions")
        pool_args = [kp.data_ptr(), vp.data_ptr(), *kp.stride()[:3], table.data_ptr(),
                     table.stride(0), kp.shape[1]]
    ld = [t.stride(0) if tokens > 1 else t.shape[1] for t in rows]
    _lib.check(
        _lib.library().lse_rope_kv(
            rows[0].data_ptr(), ld[0], rows[1].data_ptr(), ld[1], rows[2].data_ptr(), ld[2],
            rows[3].data_ptr(), rows[4].data_ptr(), ld[3], out.data_ptr(), *cache_args, *pool_args,
            n_heads, n_kv, d, sequences, ntok, start, _stream(dev)),
        "lse_rope_kv",
    )
    return out


# ---- rotary positions and the 8-bit K/V cache ----------------------------------------------------

KV_GROUP = 16  # positions of a head that share a scale
_F8, _E8, _BF16, _I32 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16, torch.int32


def _one_gpu(first: torch.Tensor, *others: torch.Tensor) -> int:
    """`_on_gpu` in one call a tensor (get_device is -1 on the host)."""
    dev = first.get_device()
    for t in others:
        if t.get_device() != dev:
            return _on_gpu(first, *others)
    return dev if dev >= 0 else _on_gpu(first)


def _launch(dev: int, what: str, args: bytes | int, *more) -> None:
    """Calls the entry point `what` with its (packed) args and dev's current stream. A kernel goes to the current
    device, whose default stream has the handle of every other's."""
    fn = getattr(_lib._lib or _lib.library(), what)
    if torch._C._cuda_getDevice() == dev:
        status = fn(args, *more, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(args, *more, torch._C._cuda_getCurrentRawStream(dev))
    if status:
        _lib.check(status, what)


# Entries of a `rope_scaling` by kind: those it needs, those it may have.
_LONG = ("factor", "original_max_position_embeddings")
_ROPE_SCALING = {
    "default": ((), ()), "linear": (("factor",), ()),
    "llama3": ((*_LONG, "low_freq_factor", "high_freq_factor"), ()),
    "yarn": (_LONG, ("beta_fast", "beta_slow", "attention_factor")),
}


def rope_table(positions: int, rotary: int, theta: float = 10000.0, scaling: dict | None = None,
               device: torch.device | str | int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin) of positions 0 .. positions - 1, each (positions, rotary / 2) fp32: what `rope` and
    `append_kv_fp8` rotate by. Angles are computed in fp64, so far positions keep their precision.

    `scaling` is a model configuration's `rope_scaling` for contexts longer than it was trained on:
    {"rope_type": "linear", "factor"}, {"rope_type": "llama3", "factor", "low_freq_factor",
    "high_freq_factor", "original_max_position_embeddings"} or {"rope_type": "yarn", "factor",
    "original_max_position_embeddings"} with yarn's optional "beta_fast", "beta_slow" and
    "attention_factor" (which multiplies cos and sin). Other entries would change the table and are refused."""
    _require(rotary >= 2 and rotary % 2 == 0, f"rotary must be even, got {rotary}")
    _require(positions >= 1, f"a table needs at least one position, got {positions}")
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _ROPE_SCALING:
        raise RuntimeError(f"unknown rope_type {kind!r}")
    needs, may = _ROPE_SCALING[kind]
    other = set(scaling) - {"rope_type", "type", "rope_theta", "partial_rotary_factor", *needs, *may}
    _require(not other, f"unknown entries of {kind} scaling: {sorted(other)}")
    _require(all(n in scaling for n in needs), f"{kind} scaling needs {needs}")
    _require(scaling.get("rope_theta", theta) == theta, f"theta is {theta}, the scaling's {scaling.get('rope_theta')}")
    pair = torch.arange(0, rotary, 2, dtype=torch.float64, device=device) / rotary
    freq = 1.0 / theta ** pair
    gain = 1.0
    if kind == "linear":
        freq = freq / scaling["factor"]
    elif kind == "llama3":
        # Wavelengths a context of `original` holds fewer than `low` times are stretched by the factor,
        # those it holds more than `high` times are kept, linear in between.
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        turns = scaling["original_max_position_embeddings"] * freq / (2.0 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = keep * freq + (1.0 - keep) * freq / scaling["factor"]
    elif kind == "yarn":
        factor, original = scaling["factor"], scaling["original_max_position_embeddings"]
        # The pair whose wavelength a context of `original` holds `turns` times.
        where = lambda turns: (rotary * math.log(original / (turns * 2.0 * math.pi))  # noqa: E731
                               / (2.0 * math.log(theta)))
        first = max(math.floor(where(scaling.get("beta_fast") or 32.0)), 0)
        last = min(math.ceil(where(scaling.get("beta_slow") or 1.0)), rotary - 1)
        index = torch.arange(rotary // 2, dtype=torch.float64, device=device)
        keep = 1.0 - ((index - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        freq = keep * freq + (1.0 - keep) * freq / factor
        gain = scaling.get("attention_factor")
        if gain is None:
            gain = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return (gain * torch.cos(angle)).float(), (gain * torch.sin(angle)).float()


def _head_rows(t: torch.Tensor, what: str) -> tuple[torch.Tensor, int, int, int]:
    """(tokens, heads, D) bf16 as rows of heads the kernels take (D contiguous, strides multiples of 8
    elements, a 16-byte aligned address): owner, address, strides of tokens and heads."""
    if t.dtype is not _BF16 or t.dim() != 3:
        raise RuntimeError(f"{what} must be a bf16 (tokens, heads, D) tensor, got {tuple(t.shape)} {t.dtype}")
    st, sh, sd = t.stride()
    at = t.data_ptr()
    if sd != 1 or (st | sh) & 7 or at & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        st, sh, _ = t.stride()
        at = t.data_ptr()
    return t, at, st, sh


def _rope_tables(cos: torch.Tensor, sin: torch.Tensor, d: int) -> tuple[int, int]:
    """(rows, rotary dims) of two tables as `rope_table` makes them, for heads of d dims."""
    if (cos.dtype is not torch.float32 or sin.dtype is not torch.float32 or cos.dim() != 2
            or cos.shape != sin.shape or not cos.is_contiguous() or not sin.is_contiguous()):
        raise RuntimeError("cos and sin must be contiguous fp32 (positions, rotary / 2) tensors")
    rows, half = cos.shape
    if half < 8 or half & 7 or 2 * half > d or d & 15:
        raise RuntimeError(f"rotary dims and D must be multiples of 16, rotary at most D; got {2 * half} of {d}")
    return rows, 2 * half


def rope(
    q: torch.Tensor, k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor,
    positions: torch.Tensor, interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """q (tokens, H, D) and k (tokens, H_KV, D) or None, bf16, rotated to `positions` (tokens,) int32, in
    one kernel: pair i of a head's first R dims, (i, i + R / 2), or (2 i, 2 i + 1) when interleaved, is turned
    by the angle whose cosine and sine are in row `positions[t]`, column i of cos and sin (`rope_table`,
    fp32, (rows, R / 2)); the dims from R on are copied. Computed in fp32, rounded once. A position outside
    the tables gives NaN. D and R are multiples of 16. Tokens and heads may be strided."""
    dev = _one_gpu(q, cos, sin, positions)
    q2, q_at, qt, qh = _head_rows(q, "q")
    tokens, h, d = q2.shape
    rows, rotary = _rope_tables(cos, sin, d)
    if positions.dtype is not _I32 or positions.shape != (tokens,):
        raise RuntimeError(f"positions must be int32 ({tokens},)")
    at = positions if positions.is_contiguous() else positions.contiguous()
    q_out = torch.empty_like(q2, memory_format=torch.contiguous_format)
    k_out, k_at, kt, kh, n_kv, k_out_at = None, 0, 0, 0, 0, 0
    if k is not None:
        _one_gpu(q, k)
        k2, k_at, kt, kh = _head_rows(k, "k")
        k_tokens, n_kv, dk = k2.shape
        if k_tokens != tokens or dk != d:
            raise RuntimeError("q and k must have the same tokens and D")
        k_out = torch.empty_like(k2, memory_format=torch.contiguous_format)
        k_out_at = k_out.data_ptr()
    _launch(dev, "lse_rope", _lib.ROPE_ARGS.pack(
        q_at, qt, qh, k_at, kt, kh, cos.data_ptr(), sin.data_ptr(), rows, at.data_ptr(), q_out.data_ptr(),
        k_out_at, tokens, h, n_kv, d, rotary, int(interleaved)))
    return q_out, k_out


class Fp8KV(NamedTuple):
    """A layer's paged K/V cache in 8 bits, in the layout its kernels stream (`fp8_kv_pool`): float8 e4m3
    codes k and v (blocks, H_KV, S, 16 D), S = block_size / 16 groups of 16 positions in a block, and their
    scales, powers of two (e8m0), (blocks, H_KV, S, 2) for k and v. `unpack_fp8_kv` gives the values."""

    k: torch.Tensor
    v: torch.Tensor
    scales: torch.Tensor

    @property
    def block_size(self) -> int:
        return KV_GROUP * self.k.shape[2]


def fp8_kv_pool(num_blocks: int, block_size: int, n_kv: int, d: int,
                device: torch.device | str | int) -> Fp8KV:
    """An 8-bit K/V pool of zeros: 1 byte per value and 1/(16 D) for the scales."""
    _require(block_size >= KV_GROUP and block_size % KV_GROUP == 0,
             f"block_size must be a multiple of {KV_GROUP}, got {block_size}")
    _require(d in (64, 128), f"D must be 64 or 128, got {d}")
    shape = (num_blocks, n_kv, block_size // KV_GROUP)
    code = lambda: torch.zeros((*shape, KV_GROUP * d), dtype=torch.uint8,  # noqa: E731
                               device=device).view(torch.float8_e4m3fn)
    scales = torch.ones((*shape, 2), dtype=torch.uint8, device=device)  # 2^-126, the least
    return Fp8KV(code(), code(), scales.view(torch.float8_e8m0fnu))


def unpack_fp8_kv(pool: Fp8KV) -> tuple[torch.Tensor, torch.Tensor]:
    """The values a pool stands for, as two bf16 (blocks, block_size, H_KV, D) tensors (the layout of
    `paged_attention_forward`'s pools; exact but for values below 2^-126, which bf16 holds in steps of 2^-133;
    done with torch operations)."""
    blocks, n_kv, per, size = pool.k.shape
    d = size // KV_GROUP
    k = pool.k.view(torch.uint8).reshape(blocks, n_kv, per, 4, d // 64, 4, 64).transpose(4, 5)
    v = pool.v.view(torch.uint8).reshape(blocks, n_kv, per, d, KV_GROUP).transpose(3, 4)
    got = []
    for what, codes in enumerate((k, v)):
        codes = codes.reshape(blocks, n_kv, per, KV_GROUP, d).contiguous().view(torch.float8_e4m3fn)
        values = codes.float() * pool.scales[..., what].float()[..., None, None]
        got.append(values.permute(0, 2, 3, 1, 4).reshape(blocks, per * KV_GROUP, n_kv, d)
                   .to(torch.bfloat16))
    return got[0], got[1]


def _check_fp8_pool(pool: Fp8KV) -> tuple[int, int, int, int, int, int]:
    """(blocks, H_KV, S, D, bytes from a block to the next in k and v, and in scales) of a pool."""
    k, v, s = pool
    shape = k.shape
    if k.dtype is not _F8 or v.dtype is not _F8 or len(shape) != 4 or v.shape != shape:
        raise RuntimeError("pool codes must be two float8_e4m3fn (blocks, H_KV, S, 16 D) tensors")
    blocks, n_kv, per, size = shape
    if s.dtype is not _E8 or s.shape != (blocks, n_kv, per, 2):
        raise RuntimeError(f"pool scales must be float8_e8m0fnu ({blocks}, {n_kv}, {per}, 2)")
    if size != 128 * KV_GROUP and size != 64 * KV_GROUP or per < 1 or n_kv < 1:
        raise RuntimeError(f"pool groups of {size} bytes: D must be 64 or 128")
    stride, s_stride = n_kv * per * size, 2 * n_kv * per
    if not (k.is_contiguous() and v.is_contiguous() and s.is_contiguous()):
        if blocks > 1:
            stride, s_stride = k.stride(0), s.stride(0)
            if v.stride(0) != stride:
                raise RuntimeError("a pool's k and v must have their blocks equally far apart")
        if not (k[:1].is_contiguous() and v[:1].is_contiguous() and s[:1].is_contiguous()):
            raise RuntimeError("a pool's blocks must be contiguous")
    return blocks, n_kv, per, size // KV_GROUP, stride, s_stride


def _check_plan(table: torch.Tensor, *entry: torch.Tensor) -> tuple[int, int, int]:
    """(entries, blocks, row stride) of a batch plan's block_table (entries, blocks); the others are int32
    (entries,) tensors."""
    if table.dtype is not _I32 or table.dim() != 2:
        raise RuntimeError(f"block_table must be an int32 (E, B) tensor, got {tuple(table.shape)} {table.dtype}")
    entries, width = table.shape
    stride, column = table.stride()
    if column != 1 and width > 1:
        raise RuntimeError("block_table must have unit column stride")
    for t in entry:
        if t.dtype is not _I32 or t.dim() != 1 or t.numel() != entries or not t.is_contiguous():
            raise RuntimeError(f"context_len, query_offset, q_start and q_len must be contiguous int32 "
                               f"({entries},) tensors")
    return entries, width, stride if entries > 1 else width


def append_kv_fp8(
    q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor | None,
    sin: torch.Tensor | None, pool: Fp8KV, block_table: torch.Tensor, query_offset: torch.Tensor,
    q_start: torch.Tensor, q_len: torch.Tensor, max_q_len: int, interleaved: bool = False,
) -> torch.Tensor | None:
    """Writes a batch plan's new k and v rows into an 8-bit paged pool, rotating q and k on the way (as
    `rope`, by the entries' positions; cos and sin None: not at all), in one kernel.

    q (tokens, H, D) or None, k and v (tokens, H_KV, D): bf16, tokens and heads may be strided. Entry e's rows
    are q_start[e] + m, m < q_len[e] <= max_q_len, at positions query_offset[e] + m of the blocks that
    block_table[e] names; entries own their rows and the blocks they write to. A group of 16 positions
    takes the smallest power-of-two scale that keeps its finite values within 448 scales; positions it held
    before are requantised when its scale grows, and slots behind the last new one are zeroed. Infinities
    and NaN are held as NaN. Positions outside the table, blocks outside the pool, entries of a negative
    query_offset and rows outside q, k and v are dropped: their k and v are not written. Returns the rotated q
    (tokens, H, D), of which rows of no entry are not written."""
    dev = _one_gpu(k, v, *pool, block_table, query_offset, q_start, q_len)
    blocks, n_kv, per, d, stride, s_stride = _check_fp8_pool(pool)
    entries, width, t_stride = _check_plan(block_table, query_offset, q_start, q_len)
    k2, k_at, kt, kh = _head_rows(k, "k")
    v2, v_at, vt, vh = _head_rows(v, "v")
    tokens, heads, dk = shape = k2.shape
    if heads != n_kv or dk != d or v2.shape != shape:
        raise RuntimeError(f"k and v must be (tokens, {n_kv}, {d}) for this pool")
    rows = rotary = cos_at = sin_at = 0
    if cos is not None and sin is not None:
        _one_gpu(k, cos, sin)
        rows, rotary = _rope_tables(cos, sin, d)
        cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
    elif cos is not sin:
        raise RuntimeError("cos and sin go together")
    h, q_at, qt, qh, q_out, out_at = n_kv, 0, 0, 0, None, 0
    if q is not None:
        _one_gpu(k, q)
        q2, q_at, qt, qh = _head_rows(q, "q")
        q_tokens, h, dq = q2.shape
        if q_tokens != tokens or dq != d or h % n_kv or h == 0:
            raise RuntimeError(f"q must be ({tokens}, H, {d}), H a multiple of {n_kv}")
        q_out = torch.empty_like(q2, memory_format=torch.contiguous_format)
        out_at = q_out.data_ptr()
    _launch(dev, "lse_append_kv_fp8", _lib.APPEND_KV_FP8_ARGS.pack(
        q_at, qt, qh, k_at, kt, kh, v_at, vt, vh, cos_at, sin_at, rows, out_at, pool.k.data_ptr(),
        pool.v.data_ptr(), stride, pool.scales.data_ptr(), s_stride, blocks, KV_GROUP * per,
        block_table.data_ptr(), t_stride, width, query_offset.data_ptr(), q_start.data_ptr(), q_len.data_ptr(),
        entries, tokens, max_q_len, h, n_kv, d, rotary, int(interleaved)))
    return q_out


def paged_attention_fp8(
    q: torch.Tensor, pool: Fp8KV, block_table: torch.Tensor, context_len: torch.Tensor,
    query_offset: torch.Tensor, q_start: torch.Tensor, q_len: torch.Tensor, max_q_len: int,
) -> torch.Tensor:
    """`paged_attention_forward` over an 8-bit pool: one call for a whole batch plan's attention at one
    layer, the same plan tensors and meaning, k and v being the values the pool stands for.

    q: (H, tokens, D) bf16, D contiguous; D = 64 or 128, 1 <= H / H_KV <= 16. block_table (entries,
    max_blocks), context_len, query_offset, q_start, q_len (entries,): int32 on the device; entries own
    distinct rows of q; max_q_len >= every q_len. Returns o like q; rows of no entry are not written. Softmax
    scale 1/sqrt(D)."""
    dev = _one_gpu(q, *pool, block_table, context_len, query_offset, q_start, q_len)
    blocks, n_kv, per, d, stride, s_stride = _check_fp8_pool(pool)
    entries, width, t_stride = _check_plan(block_table, context_len, query_offset, q_start, q_len)
    if q.dim() != 3 or q.dtype is not _BF16:
        raise RuntimeError(f"q must be bf16 (H, tokens, {d}) with a contiguous head dim")
    h, tokens, dq = q.shape
    sh, st, sd = q.stride()
    if dq != d or sd != 1:
        raise RuntimeError(f"q must be bf16 (H, tokens, {d}) with a contiguous head dim")
    if h == 0 or h % n_kv or h // n_kv > 16:
        raise RuntimeError(f"unsupported attention shape: H={h} H_KV={n_kv} D={d}")
    o = torch.empty_like(q)
    oh, ot, _ = o.stride()
    args = _lib.PAGED_ATTENTION_FP8_ARGS.pack(
        q.data_ptr(), sh, st, pool.k.data_ptr(), pool.v.data_ptr(), stride, pool.scales.data_ptr(), s_stride,
        blocks, KV_GROUP * per, block_table.data_ptr(), t_stride, width, context_len.data_ptr(),
        query_offset.data_ptr(), q_start.data_ptr(), q_len.data_ptr(), o.data_ptr(), oh, ot, entries, tokens,
        max_q_len, h, n_kv, d, d ** -0.5)
    nbytes = (_lib._lib or _lib.library()).lse_paged_attention_fp8_workspace_bytes(args)
    if nbytes < 0:
        raise RuntimeError(f"unsupported attention sizes: max_q_len={max_q_len}, {width} blocks of "
                           f"{KV_GROUP * per}")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _launch(dev, "lse_paged_attention_fp8", args, *_ws_args(ws))
    return o


def packed_bf16_shape(n: int, k: int) -> tuple[int, int, int]:
    return ((n + 15) // 16, (k + 63) // 64, 1024)


def pack_bf16_weight(w: torch.Tensor) -> torch.Tensor:
    """Row-major (N, K) bf16 → the bf16 tile layout, a (ceil(N/16), ceil(K/64), 1024) bf16
    tensor (2 KB per 16-row x 64-K step: the lo and hi MFMA operands), on the GPU."""
    _require(w.dim() == 2 and w.dtype == torch.bfloat16, "w must be a 2-D bf16 tensor")
    dev = _on_gpu(w)
    n, k = w.shape
    w2 = w if w.stride(1) == 1 and w.stride(0) % 8 == 0 and w.data_ptr() % 16 == 0 else w.contiguous()
    wp = torch.empty(packed_bf16_shape(n, k), dtype=torch.bfloat16, device=dev)
    _lib.check(_lib.library().lse_pack_bf16_weight(w2.data_ptr(), w2.stride(0), n, k,
                                                    wp.data_ptr(), _stream(dev)),
               "lse_pack_bf16_weight")
    return wp


def unpack_bf16_weight(wp: torch.Tensor, n: int, k: int) -> torch.Tensor:
    """Inverse of `pack_bf16_weight` (a pure permutation, done with torch views): (N, K) bf16."""
    rb, steps, _ = wp.shape
    t = wp.reshape(rb, steps, 2, 4, 16, 8)  # [rb][step][half][g = lane // 16][row][8 elements]
    t = t.permute(0, 4, 1, 3, 2, 5).reshape(rb * 16, steps * 64)
    return t[:n, :k].contiguous()


def bf16_decode_linear(x: torch.Tensor, wp: torch.Tensor, n: int) -> torch.Tensor:
    """y = bf16(x · wᵀ) for x (..., K) bf16, w given packed (`pack_bf16_weight`) → y (..., N)
    bf16; fp32 accumulation. Built for decode batches (the decode kernel up to 16 rows, bf16
    tiles of the tiled kernel above), correct for any number of rows."""
    dev = _on_gpu(x, wp)
    if x.dtype is not torch.bfloat16:
        raise RuntimeError(f"expects bf16 activations, got {x.dtype}")
    lead = x.shape
    k = lead[-1]
    if wp.dtype is not torch.bfloat16 or wp.shape != packed_bf16_shape(n, k):
        raise RuntimeError(f"packed weight has shape {tuple(wp.shape)}, (N, K) = ({n}, {k}) needs "
                           f"{packed_bf16_shape(n, k)}")
    owner, at, ldx, m = _row_args(x, k)
    y = torch.empty((*lead[:-1], n), dtype=torch.bfloat16, device=dev)
    _lib.check(
        _lib.library().lse_bf16_decode_gemm(at, ldx, wp.data_ptr(), y.data_ptr(), n, m, n, k,
                                            _stream(dev)),
        "lse_bf16_decode_gemm",
    )
    return y


# ---- 4-bit weights, and rows in 8 bits -----------------------------------------------------------

FP4_GROUP = 32  # weights of a row, or values of a row in 8 bits, that share a scale
FP4_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # of the e2m1 codes 0 to 7; 8 more is the sign


class Fp4Weight(NamedTuple):
    """A 4-bit weight in the tiles that the products stream: float4 e2m1 codes with a power of two (e8m0) for every
    32 consecutive k of a row.

    codes: uint8 (tiles, ceil(K / 128), 1024), scales: float8_e8m0fnu, or its bytes as uint8, (tiles, ceil(K / 512),
    256); n: the columns of the product, k: those of its input. tiles = ceil(n / 16); 2 ceil(n / 16) for the gate and up
    weights of a `w4a16_glu` or `w4a8_glu`, whose row tiles take turns. Made by `pack_fp4`."""

    codes: torch.Tensor
    scales: torch.Tensor
    n: int
    k: int


class Fp8Rows(NamedTuple):
    """Rows held in 8 bits: float8 e4m3 codes (..., K) and a power of two (e8m0) for every 32 of a row's values,
    scales (..., K / 32). Made by `quantize_rows_fp8` and `add_rmsnorm_fp8`."""

    codes: torch.Tensor
    scales: torch.Tensor


def quantize_weight_fp4(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """W (N, K) → codes uint8 (N, K / 2), two e2m1 codes a byte with the lower k in the low half, and scales
    float8_e8m0fnu (N, K / 32): the smallest power of two from 2^-126 up that has its 32 weights within 6 scales;
    each weight goes to the nearest code, ties to the even one. A group with a value that is not finite gets the scale
    NaN. K % 32 == 0. Runs on the GPU at load time; W is read as fp32 (bf16 and fp16 widen exactly)."""
    _require(w.dim() == 2 and w.is_floating_point(), f"weight must be 2-D floating point, got {tuple(w.shape)} {w.dtype}")
    dev = _on_gpu(w)
    n, k = w.shape
    _require(k % FP4_GROUP == 0, f"4-bit weights need K % {FP4_GROUP} == 0, got K = {k}")
    w32 = w.to(torch.float32).contiguous()
    if w32.data_ptr() % 16:
        w32 = w32.clone()
    codes = torch.empty((n, k // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty((n, k // FP4_GROUP), dtype=_E8, device=dev)
    _launch(dev, "lse_quantize_weight_fp4", w32.data_ptr(), k, codes.data_ptr(), scales.data_ptr(), n, k)
    return codes, scales


def _check_fp4_rows(codes: torch.Tensor, scales: torch.Tensor) -> tuple[int, int]:
    """(rows, K) of a weight's codes and scales row by row."""
    if codes.dim() != 2 or codes.dtype is not torch.uint8 or scales.dim() != 2 or scales.dtype is not _E8:
        raise RuntimeError("codes must be uint8 (N, K / 2), scales float8_e8m0fnu (N, K / 32)")
    n, k = codes.shape[0], 2 * codes.shape[1]
    if k % FP4_GROUP or scales.shape != (n, k // FP4_GROUP):
        raise RuntimeError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are no 4-bit weight")
    return n, k


def pack_fp4(codes: torch.Tensor, scales: torch.Tensor, glu: bool = False) -> Fp4Weight:
    """A 4-bit weight row by row (`quantize_weight_fp4`'s form) → its tiles, on the GPU. glu: the rows are (2 I, K)
    [gate; up], for `w4a16_glu` and `w4a8_glu`; n is then I."""
    dev = _on_gpu(codes, scales)
    rows, k = _check_fp4_rows(codes, scales)
    _require(not glu or rows % 2 == 0, "gate and up rows come in equal numbers")
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 16:
        codes = codes.clone()
    n = rows // 2 if glu else rows
    tiles = -(-n // 16) * (2 if glu else 1)
    out = Fp4Weight(torch.empty((tiles, -(-k // 128), 1024), dtype=torch.uint8, device=dev),
                    torch.empty((tiles, -(-k // 512), 256), dtype=_E8, device=dev), n, k)
    _launch(dev, "lse_pack_fp4", codes.data_ptr(), scales.data_ptr(), out.codes.data_ptr(), out.scales.data_ptr(), rows,
            k, int(glu))
    return out


def unpack_fp4(weight: Fp4Weight) -> tuple[torch.Tensor, torch.Tensor]:
    """Inverse of `pack_fp4` (a pure permutation, done with torch views): (codes, scales) row by row."""
    _, tiles = _check_fp4(weight, None)
    glu, n, k = tiles != -(-weight.n // 16), weight.n, weight.k
    steps, chunks = weight.codes.shape[1], weight.scales.shape[1]
    c = weight.codes.view(tiles, steps, 4, 16, 16).permute(0, 3, 1, 2, 4).reshape(tiles * 16, 64 * steps)[:, :k // 2]
    s = weight.scales.view(torch.uint8).view(tiles, chunks, 4, 16, 4).permute(0, 3, 1, 4, 2)
    s = s.reshape(tiles * 16, 16 * chunks)[:, :k // FP4_GROUP]
    if glu:
        c, s = (t.reshape(tiles // 2, 2, 16, t.shape[1]).transpose(0, 1).reshape(2, tiles * 8, t.shape[1])[:, :n]
                .flatten(0, 1) for t in (c, s))
    else:
        c, s = c[:n], s[:n]
    return c.contiguous(), s.contiguous().view(_E8)


def dequantize_fp4(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The values of a 4-bit weight row by row, (N, K) fp32."""
    n, k = _check_fp4_rows(codes, scales)
    value = torch.tensor([*FP4_MAGNITUDES, *(-v for v in FP4_MAGNITUDES)], device=codes.device)
    w = value[torch.stack([codes & 15, codes >> 4], -1).view(n, k).int()]
    return (w.view(n, k // FP4_GROUP, FP4_GROUP) * scales.float()[..., None]).view(n, k)


def dequantize_rows_fp8(rows: Fp8Rows) -> torch.Tensor:
    """The values of rows in 8 bits, (..., K) bf16: exact, but that the two smallest scales have values below
    bf16's subnormals, which round to them."""
    v = rows.codes.float().unflatten(-1, (-1, FP4_GROUP)) * rows.scales.float()[..., None]
    return v.flatten(-2).to(_BF16)


# Allocations cost a decode call more than its checks, so they take the cheapest way there is: a tensor like another
# (1.1 us), by size and stride (1.3), by shape (1.6 to 2.2).


def _empty_2d(lead: torch.Size, n: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """An uninitialised contiguous (*lead, n)."""
    if len(lead) == 1:
        return torch.empty_strided((lead[0], n), (n, 1), dtype=dtype, device=device)
    return torch.empty((*lead, n), dtype=dtype, device=device)


def _empty_rows(x: torch.Tensor, k: int) -> tuple[Fp8Rows, int]:
    """Rows in 8 bits for x (..., K), and the bytes from a row's scales to the next: the products read whole dwords."""
    per = k // FP4_GROUP
    lds = (per + 3) & ~3
    codes = torch.empty_like(x, dtype=_F8) if x.is_contiguous() else torch.empty(x.shape, dtype=_F8, device=x.device)
    scales = _empty_2d(x.shape[:-1], lds, _E8, x.device)
    return Fp8Rows(codes, scales if lds == per else scales[..., :per]), lds


def quantize_rows_fp8(x: torch.Tensor) -> Fp8Rows:
    """x (..., K) bf16 → its rows in 8 bits: for every 32 values of a row the smallest power of two from 2^-126 up that
    has the finite ones within 448 scales, and their codes, rounded to nearest even (none to 2^128; infinity and NaN
    become NaN). K % 32 == 0."""
    dev = _one_gpu(x)
    if x.dtype is not _BF16:
        raise RuntimeError(f"rows in 8 bits are made of bf16 rows, got {x.dtype}")
    k = x.shape[-1]
    if k % FP4_GROUP:
        raise RuntimeError(f"rows in 8 bits need K % {FP4_GROUP} == 0, got K = {k}")
    owner, at, ldx, m = _row_args(x, k) if k else (x, 0, 0, 0)
    rows, lds = _empty_rows(x, k)
    _launch(dev, "lse_quantize_rows_fp8", at, ldx, rows.codes.data_ptr(), rows.scales.data_ptr(), lds, m, k)
    return rows


def add_rmsnorm_fp8(
    x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float,
) -> tuple[torch.Tensor, Fp8Rows]:
    """(s, LlamaRMSNorm(s) in 8 bits) with s = x + residual (x itself when residual is None) in one kernel: `add_rmsnorm`
    and `quantize_rows_fp8` after it, but that the mean and its root are held in 64 bits. x and residual (..., K) bf16,
    weight (K,) bf16, K % 32 == 0, K <= `_lib.NORM_MAX_K`."""
    dev = _one_gpu(x, weight) if residual is None else _one_gpu(x, weight, residual)
    k = x.shape[-1]
    if x.dtype is not _BF16 or weight.dtype is not _BF16 or weight.shape != (k,):
        raise RuntimeError(f"RMSNorm takes bf16 x and weight ({k},)")
    if k % FP4_GROUP or k > _lib.NORM_MAX_K or k == 0:
        raise RuntimeError(f"a norm into 8 bits needs K % {FP4_GROUP} == 0 up to {_lib.NORM_MAX_K}, got K = {k}")
    owner, at, ldx, m = _row_args(x, k)
    s, r_at, ldr, s_at = x, 0, 0, 0
    if residual is not None:
        if residual.dtype is not _BF16 or residual.shape != x.shape:
            raise RuntimeError("the residual must be bf16 and of x's shape")
        r_owner, r_at, ldr, _ = _row_args(residual, k)
        s = torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=_BF16, device=x.device)
        s_at = s.data_ptr()
    w = weight.contiguous()
    if w.data_ptr() % 16:  # a piece of a flat parameter buffer
        w = w.clone()
    rows, lds = _empty_rows(x, k)
    _launch(dev, "lse_add_rmsnorm_fp8", _lib.ADD_RMSNORM_FP8_ARGS.pack(
        at, ldx, r_at, ldr, w.data_ptr(), s_at, rows.codes.data_ptr(), rows.scales.data_ptr(), lds, m, k, float(eps)))
    return s, rows


def _check_fp4(weight: Fp4Weight, glu: bool | None) -> tuple[int, int]:
    """(n, tiles) of a 4-bit weight, its tiles checked; glu None: of either kind."""
    codes, scales, n, k = weight
    tiles = codes.shape[0]
    if (codes.dtype is not torch.uint8 or scales.dtype not in (_E8, torch.uint8) or not codes.is_contiguous()
            or not scales.is_contiguous() or (codes.data_ptr() | scales.data_ptr()) % 16):
        raise RuntimeError("a 4-bit weight's codes must be uint8 and its scales float8_e8m0fnu, contiguous, 16-byte "
                           "aligned")
    if k % FP4_GROUP or codes.shape != (tiles, -(-k // 128), 1024) or scales.shape != (tiles, -(-k // 512), 256):
        raise RuntimeError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are no tiles of K = {k}")
    once = -(-n // 16)
    if tiles != (2 * once if glu else once) and not (glu is None and tiles == 2 * once):
        raise RuntimeError(f"{tiles} row tiles are no {'gate/up ' if glu else ''}weight of n = {n}")
    return n, tiles


def _dword_rows(scales: torch.Tensor, per: int) -> tuple[torch.Tensor, int]:
    """Scales (M, per) whose rows start at, and may be read to, a whole dword, and the bytes from row to row: as they are
    where they allow it."""
    m, whole = scales.shape[0], (per + 3) & ~3
    lds = scales.stride(0) if m > 1 else whole
    if (scales.stride(1) != 1 or lds % 4 or not whole <= lds <= _lib.FP4_MAX_K or scales.data_ptr() % 4
            or (whole != per and scales.storage_offset() + (m - 1) * lds + whole > scales.untyped_storage().nbytes())):
        rows = torch.empty((m, whole), dtype=_E8, device=scales.device)
        rows[:, :per] = scales
        return rows, whole
    return scales, lds


def _fp8_row_args(rows: Fp8Rows, k: int):
    """(owners, codes' address and row stride, scales' address and row stride, rows) of rows in 8 bits; the owners are to
    be kept until the kernel is enqueued."""
    codes, scales = rows
    per = k // FP4_GROUP
    if codes.dtype is not _F8 or scales.dtype is not _E8:
        raise RuntimeError(f"rows in 8 bits are float8_e4m3fn with float8_e8m0fnu scales, got {codes.dtype}, "
                           f"{scales.dtype}")
    shape = codes.shape
    if shape[-1] != k or scales.shape != (*shape[:-1], per):
        raise RuntimeError(f"rows {tuple(shape)} with scales {tuple(scales.shape)} do not fit K = {k}")
    at, s_at = codes.data_ptr(), scales.data_ptr()
    if per % 4 == 0 and at % 16 == 0 and s_at % 4 == 0 and codes.is_contiguous() and scales.is_contiguous():
        return rows, at, k, s_at, per, codes.numel() // k
    codes, scales = codes.reshape(-1, k), scales.reshape(-1, per)
    m = codes.shape[0]
    ldx = codes.stride(0) if m > 1 else k
    if codes.stride(1) != 1 or not k <= ldx <= _lib.FP4_MAX_K or ldx % 16 or codes.data_ptr() % 16:
        codes, ldx = codes.clone(memory_format=torch.contiguous_format), k
    scales, lds = _dword_rows(scales, per)
    return (codes, scales), codes.data_ptr(), ldx, scales.data_ptr(), lds, m


def _fp4_gemm(x: torch.Tensor | Fp8Rows, weight: Fp4Weight, glu: bool) -> torch.Tensor:
    _check_fp4(weight, glu)
    codes, scales, n, k = weight
    if k == 0:
        raise RuntimeError("a product needs K > 0")
    if isinstance(x, Fp8Rows):
        dev = _one_gpu(codes, scales, *x)
        lead = x.codes.shape[:-1]
        owner, at, ldx, s_at, lds, m = _fp8_row_args(x, k)
    else:
        dev = _one_gpu(codes, scales, x)
        if x.dtype is not _BF16:
            raise RuntimeError(f"expected bf16 rows or Fp8Rows, got {x.dtype}")
        lead = x.shape[:-1]
        owner, at, ldx, m = _row_args(x, k)
        if ldx > _lib.FP4_MAX_K:
            owner = owner.contiguous()
            at, ldx = owner.data_ptr(), k
        s_at = lds = 0
    y = _empty_2d(lead, n, _BF16, codes.device)
    args = _lib.FP4_GEMM_ARGS.pack(at, ldx, s_at, lds, codes.data_ptr(), scales.data_ptr(), y.data_ptr(), n, m, n, k, glu)
    nbytes = (_lib._lib or _lib.library()).lse_fp4_gemm_workspace_bytes(args)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=y.device) if nbytes > 0 else None
    _launch(dev, "lse_fp4_gemm", args, *_ws_args(ws))
    return y


def w4a16_linear(x: torch.Tensor, weight: Fp4Weight) -> torch.Tensor:
    """y = bf16(sum_k x[..., k] w[n, k]) for x (..., K) bf16 → y (..., N) bf16: exact products with the 4-bit weight's
    values, fp32 sums."""
    if isinstance(x, Fp8Rows):
        raise RuntimeError("rows in 8 bits go to w4a8_linear")
    return _fp4_gemm(x, weight, False)


def w4a16_glu(x: torch.Tensor, weight: Fp4Weight) -> torch.Tensor:
    """h = silu(x Gᵀ) * (x Uᵀ) for x (..., K) bf16 and stacked 4-bit weights (`pack_fp4(..., glu=True)`) → (..., I)
    bf16, rounded once."""
    if isinstance(x, Fp8Rows):
        raise RuntimeError("rows in 8 bits go to w4a8_glu")
    return _fp4_gemm(x, weight, True)


def w4a8_linear(rows: Fp8Rows, weight: Fp4Weight) -> torch.Tensor:
    """`w4a16_linear` over rows in 8 bits, at twice the matrix cores' rate."""
    if not isinstance(rows, Fp8Rows):
        raise RuntimeError("w4a8_linear takes Fp8Rows (quantize_rows_fp8, add_rmsnorm_fp8)")
    return _fp4_gemm(rows, weight, False)


def w4a8_glu(rows: Fp8Rows, weight: Fp4Weight) -> torch.Tensor:
    """`w4a16_glu` over rows in 8 bits, at twice the matrix cores' rate."""
    if not isinstance(rows, Fp8Rows):
        raise RuntimeError("w4a8_glu takes Fp8Rows (quantize_rows_fp8, add_rmsnorm_fp8)")
    return _fp4_gemm(rows, weight, True)
