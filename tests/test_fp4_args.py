"""Refusals of the 4-bit entry points, without a GPU: every call below is turned down before any HIP call is made."""

from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

FAKE = 1 << 20  # a 256-byte-aligned device address that is never used
E_NULL, E_SHAPE, E_ALIGN, E_RANGE, E_WORKSPACE = -1, -2, -3, -4, -6

GEMM = dict(x=FAKE, x_stride=4096, x_scales=None, s_stride=0, codes=FAKE, scales=FAKE, y=FAKE, y_stride=512, m=4, n=512,
            k=4096, glu=0)
ROWS8 = dict(x_scales=FAKE, s_stride=128)
NORM = dict(x=FAKE, x_stride=4096, residual=FAKE, r_stride=4096, weight=FAKE, sum=FAKE, codes=FAKE, scales=FAKE,
            s_stride=128, m=4, k=4096, eps=1e-5)


def _gemm_args(changes):
    from llm_serving_engine_amd import _lib

    assert set(changes) <= set(GEMM)
    return _lib.FP4_GEMM_ARGS.pack(*(0 if v is None else v for v in {**GEMM, **changes}.values()))


def _gemm(pkg, changes, ws=None, ws_bytes=0):
    return pkg.library().lse_fp4_gemm(_gemm_args(changes), ws, ws_bytes, None)


def _norm(pkg, changes):
    from llm_serving_engine_amd import _lib

    assert set(changes) <= set(NORM)
    args = _lib.ADD_RMSNORM_FP8_ARGS.pack(*(0 if v is None else v for v in {**NORM, **changes}.values()))
    return pkg.library().lse_add_rmsnorm_fp8(args, None)


def test_the_structs_are_the_headers(pkg):
    """As many fields as the header's structs have, each of eight bytes."""
    from llm_serving_engine_amd import _lib

    text = (Path(__file__).resolve().parent.parent / "include" / "lse_int8.h").read_text()
    for name, layout, base in (("lse_fp4_gemm_args", _lib.FP4_GEMM_ARGS, GEMM),
                               ("lse_add_rmsnorm_fp8_args", _lib.ADD_RMSNORM_FP8_ARGS, NORM)):
        body = re.search(r"struct " + name + r" \{(.*?)\};", text, re.S).group(1)
        fields = 0
        for line in body.split(";"):
            line = line.strip()
            if line:
                assert re.match(r"(const )?void( ?\*)|int64_t |double ", line), line
                fields += line.count(",") + 1
        assert fields == len(base) and layout.size == 8 * fields
    assert re.search(r"#define LSE_FP4_MAX_K (\d+)", text).group(1) == str(_lib.FP4_MAX_K)


@pytest.mark.parametrize("changes,status", [
    (dict(m=-1), E_SHAPE), (dict(n=-1), E_SHAPE), (dict(k=-32), E_SHAPE), (dict(glu=2), E_SHAPE),
    (dict(m=1 << 31), E_SHAPE), (dict(n=1 << 31), E_SHAPE), (dict(k=4080), E_ALIGN), (dict(k=0), E_RANGE),
    (dict(k=1 << 22, x_stride=1 << 22), E_RANGE), (dict(x=None), E_NULL), (dict(codes=None), E_NULL),
    (dict(scales=None), E_NULL), (dict(y=None), E_NULL), (dict(x_stride=4088), E_SHAPE), (dict(y_stride=511), E_SHAPE),
    (dict(x_stride=4100), E_ALIGN), (dict(x=FAKE + 8), E_ALIGN), (dict(codes=FAKE + 8), E_ALIGN),
    (dict(scales=FAKE + 4), E_ALIGN), (dict(y=FAKE + 1), E_ALIGN), (dict(x_stride=1 << 22), E_RANGE),
    (dict(ROWS8, s_stride=127), E_SHAPE), (dict(ROWS8, s_stride=130), E_ALIGN), (dict(ROWS8, x_scales=FAKE + 2), E_ALIGN),
    (dict(ROWS8, x_stride=4104), E_ALIGN), (dict(ROWS8, s_stride=1 << 22), E_RANGE),
    (dict(m=0, x=None), 0), (dict(n=0, y_stride=0, y=None), 0),
])
def test_gemm(pkg, changes, status):
    assert _gemm(pkg, changes) == status
    if status == E_SHAPE and "glu" not in changes and not {"x_stride", "y_stride", "s_stride"} & set(changes):
        assert pkg.library().lse_fp4_gemm_workspace_bytes(_gemm_args(changes)) == -1


def test_null_structs(pkg):
    lib = pkg.library()
    assert lib.lse_fp4_gemm(None, None, 0, None) == E_NULL and lib.lse_add_rmsnorm_fp8(None, None) == E_NULL
    assert lib.lse_fp4_gemm_workspace_bytes(None) == -1


def test_workspaces(pkg):
    """Calls whose K is split need their sums' bytes, others nothing; a missing or crooked one is refused."""
    need = lambda **c: pkg.library().lse_fp4_gemm_workspace_bytes(_gemm_args(c))  # noqa: E731
    for m in (1, 4, 16, 4096):
        assert need(m=m, n=28672, y_stride=28672) == 0
    split = dict(m=200, n=4096, y_stride=4096, k=14336, x_stride=14336)
    nbytes = need(**split)
    assert nbytes > 0 and nbytes % (200 * 4096 * 4) == 0
    assert _gemm(pkg, split) == E_WORKSPACE
    assert _gemm(pkg, split, FAKE, nbytes - 1) == E_WORKSPACE and _gemm(pkg, split, FAKE + 8, nbytes) == E_WORKSPACE
    for m in range(1, 3000, 61):
        for n in (16, 100, 1024, 4096, 28672):
            for k in (32, 512, 4096, 14336):
                for extra in ({}, ROWS8):
                    for glu in (0, 1):
                        got = need(m=m, n=n, k=k, glu=glu, **extra)
                        assert 0 <= got <= 64 << 20


@pytest.mark.parametrize("changes,status", [
    (dict(m=-1), E_SHAPE), (dict(m=1 << 31), E_SHAPE), (dict(k=4080), E_ALIGN), (dict(k=16416, x_stride=16416), E_RANGE),
    (dict(x=None), E_NULL), (dict(weight=None), E_NULL), (dict(codes=None), E_NULL), (dict(scales=None), E_NULL),
    (dict(x_stride=4064), E_SHAPE), (dict(r_stride=4064), E_SHAPE), (dict(s_stride=127), E_SHAPE), (dict(eps=-1.0), E_SHAPE),
    (dict(eps=float("nan")), E_SHAPE), (dict(x_stride=4100), E_ALIGN), (dict(r_stride=4100), E_ALIGN),
    (dict(x=FAKE + 8), E_ALIGN), (dict(residual=FAKE + 8), E_ALIGN), (dict(weight=FAKE + 8), E_ALIGN),
    (dict(sum=FAKE + 8), E_ALIGN), (dict(codes=FAKE + 8), E_ALIGN), (dict(m=0, x=None), 0),
])
def test_norm(pkg, changes, status):
    assert _norm(pkg, changes) == status


def test_rows_and_weights(pkg):
    lib = pkg.library()
    rows = lambda x=FAKE, ldx=64, c=FAKE, s=FAKE, ss=2, m=3, k=64: lib.lse_quantize_rows_fp8(x, ldx, c, s, ss, m, k, None)  # noqa: E731
    assert rows(m=-1) == rows(ldx=32) == rows(ss=1) == E_SHAPE
    assert rows(k=48) == rows(ldx=68) == rows(x=FAKE + 8) == rows(c=FAKE + 8) == E_ALIGN
    assert rows(x=None) == rows(c=None) == rows(s=None) == E_NULL
    assert rows(m=0, x=None) == 0 and rows(k=1 << 22, ldx=1 << 22, ss=1 << 17) == E_RANGE
    quant = lambda w=FAKE, ld=64, c=FAKE, s=FAKE, n=3, k=64: lib.lse_quantize_weight_fp4(w, ld, c, s, n, k, None)  # noqa: E731
    assert quant(n=-1) == quant(ld=32) == E_SHAPE and quant(k=48) == quant(ld=66) == quant(w=FAKE + 4) == E_ALIGN
    assert quant(w=None) == quant(c=None) == E_NULL and quant(n=0, w=None) == 0 and quant(k=1 << 22, ld=1 << 22) == E_RANGE
    pack = lambda c=FAKE, s=FAKE, oc=FAKE, os=FAKE, n=32, k=64, g=0: lib.lse_pack_fp4(c, s, oc, os, n, k, g, None)  # noqa: E731
    assert pack(n=-1) == pack(g=2) == pack(n=33, g=1) == E_SHAPE and pack(k=48) == pack(c=FAKE + 8) == E_ALIGN
    assert pack(c=None) == pack(os=None) == E_NULL and pack(n=0, c=None) == 0
    assert lib.lse_fp4_codes_bytes(100, 544, 0) == 7 * 5 * 1024 and lib.lse_fp4_scales_bytes(100, 544, 0) == 7 * 2 * 256
    assert lib.lse_fp4_codes_bytes(100, 544, 1) == 8 * 5 * 1024 and lib.lse_fp4_scales_bytes(100, 544, 1) == 8 * 2 * 256
    assert lib.lse_fp4_codes_bytes(99, 544, 1) == lib.lse_fp4_codes_bytes(4, 40, 0) == lib.lse_fp4_scales_bytes(-1, 32, 0) == -1


def _weight(pkg, n=32, k=128, glu=False):
    tiles = -(-n // 16) * (2 if glu else 1)
    return pkg.ops.Fp4Weight(torch.zeros(tiles, -(-k // 128), 1024, dtype=torch.uint8),
                             torch.zeros(tiles, -(-k // 512), 256, dtype=torch.uint8), n, k)


def test_python_refusals(pkg):
    """The wrappers' own checks, on tensors of the host (which they refuse last)."""
    ops, w = pkg.ops, _weight(pkg)
    x = torch.zeros(3, 128, dtype=torch.bfloat16)
    rows = ops.Fp8Rows(torch.zeros(3, 128).to(torch.float8_e4m3fn), torch.ones(3, 4).to(torch.float8_e8m0fnu))
    for call, text in (
        (lambda: ops.w4a16_linear(x, w), "CUDA"),
        (lambda: ops.w4a16_linear(rows, w), "w4a8_linear"), (lambda: ops.w4a16_glu(rows, w), "w4a8_glu"),
        (lambda: ops.w4a8_linear(x, w), "Fp8Rows"), (lambda: ops.w4a8_glu(x, w), "Fp8Rows"),
        (lambda: ops.w4a16_glu(x, w), "gate/up"), (lambda: ops.w4a16_linear(x, _weight(pkg, glu=True)), "row tiles"),
        (lambda: ops.w4a16_linear(x, w._replace(k=160)), "no tiles"), (lambda: ops.w4a16_linear(x, w._replace(k=100)), "no tiles"),
        (lambda: ops.w4a16_linear(x, w._replace(n=64)), "row tiles"),
        (lambda: ops.w4a16_linear(x, w._replace(codes=w.codes.float())), "uint8"),
        (lambda: ops.w4a16_linear(x, w._replace(scales=w.scales.float())), "e8m0"),
        (lambda: ops.quantize_rows_fp8(x), "CUDA"), (lambda: ops.quantize_weight_fp4(x), "CUDA"),
        (lambda: ops.quantize_weight_fp4(torch.zeros(4)), "2-D"), (lambda: ops.quantize_weight_fp4(torch.zeros(4, 32).int()), "floating"),
        (lambda: ops.add_rmsnorm_fp8(x, None, torch.zeros(128, dtype=torch.bfloat16), 1e-5), "CUDA"),
        (lambda: ops.pack_fp4(torch.zeros(4, 16, dtype=torch.uint8), torch.ones(4, 1).to(torch.float8_e8m0fnu)), "CUDA"),
        (lambda: ops.dequantize_fp4(torch.zeros(4, 20, dtype=torch.uint8), torch.ones(4, 1).to(torch.float8_e8m0fnu)), "no 4-bit"),
    ):
        with pytest.raises(RuntimeError, match=text):
            call()
    with pytest.raises(ValueError, match="mode"):
        pkg.Fp4Linear(64, 16, "w8a8")
    with pytest.raises(ValueError, match="multiple of 32"):
        pkg.Fp4Linear(48, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.Fp4Linear.from_linear(torch.nn.Linear(64, 16))
    for mode in ("w4a16", "w4a8"):
        pkg.ModelConfig(quantize=mode, dtype="bfloat16").validate_quantize()
        with pytest.raises(RuntimeError, match="bfloat16"):
            pkg.ModelConfig(quantize=mode).validate_quantize()


def test_unpacking_inverts_the_oracles_tiles(pkg):
    from oracle import fp4 as ora

    for n, k, glu in ((40, 544, False), (16, 32, False), (70, 1184, True), (4, 128, True)):
        g = torch.Generator().manual_seed(n)
        code, byte = torch.randint(0, 16, (n, k), generator=g), torch.randint(0, 256, (n, k // 32), generator=g)
        codes, scales = ora.tiles(code, byte, glu)
        back = pkg.ops.unpack_fp4(pkg.ops.Fp4Weight(codes, scales, n // 2 if glu else n, k))
        assert torch.equal(back[0], ora.two_a_byte(code)) and torch.equal(back[1].view(torch.uint8), byte.to(torch.uint8))
