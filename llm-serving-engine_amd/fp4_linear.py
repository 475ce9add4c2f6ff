"""`Fp4Linear` and its like: the modules of int8_linear.py over 4-bit weights, for the switch values "w4a16" and "w4a8".

They stand in the same places: `Fp4Linear` for the projections that the reference calls as modules
(src/llm_serving_engine/model/model_runner.py:322-324, 369, 418), `Fp4GluMLP` for the whole `LlamaMLP`
(transformers modeling_llama.py:163-176), `Fp8RMSNorm` for a decoder layer's two norms (modeling_llama.py:53-67).
Weights are float4 e2m1 codes with a power of two for every 32 of a row (`ops.quantize_weight_fp4`), held as the tiles
that the kernels stream (`ops.pack_fp4`); both are buffers of bytes, so `model.dtype` stays bf16 and a change of the
model's dtype leaves them alone. "w4a16" multiplies bf16 rows, "w4a8" rows in 8 bits (float8 e4m3 with a power of two
for every 32 values), which the norms make once for all projections that read them and the other projections make
themselves.
"""

from __future__ import annotations

import torch
from torch import nn

from . import ops
from .int8_linear import QKVGroup, QuantizedRows, _is_silu, group_qkv_as

MODES = ("w4a16", "w4a8")


def check_fp4_supported(linear: nn.Linear) -> None:
    """Load-time checks, raising RuntimeError as `check_linear_supported` does."""
    if linear.weight.device.type != "cuda":
        raise RuntimeError(f"4-bit kernels need a CUDA (HIP) device, got {linear.weight.device}")
    if linear.in_features == 0 or linear.in_features % ops.FP4_GROUP:
        raise RuntimeError(f"4-bit kernels need in_features % {ops.FP4_GROUP} == 0, got {linear.in_features}")


def _check_mode(mode: str) -> None:
    if mode not in MODES:
        raise ValueError(f"mode must be one of {MODES}, got {mode!r}")


def _fp8_input(mode: str, x: torch.Tensor | QuantizedRows) -> torch.Tensor | ops.Fp8Rows:
    """What the kernels take of a module's input: bf16 rows, or in "w4a8" rows in 8 bits."""
    if isinstance(x, QuantizedRows):
        if mode != "w4a8" or x.xq.dtype != torch.float8_e4m3fn:
            raise RuntimeError(f"rows of {x.xq.dtype} reach a {mode} projection")
        return ops.Fp8Rows(x.xq, x.sx)
    return ops.quantize_rows_fp8(x) if mode == "w4a8" else x


def _fp4_product(mode: str, x: torch.Tensor | QuantizedRows, qweight: torch.Tensor, scales: torch.Tensor,
                 n: int, k: int) -> torch.Tensor:
    x = _fp8_input(mode, x)
    weight = ops.Fp4Weight(qweight, scales, n, k)
    return ops.w4a8_linear(x, weight) if mode == "w4a8" else ops.w4a16_linear(x, weight)


class Fp4Linear(nn.Module):
    """y = x · Wᵀ (+ bias) with W in 4 bits. `mode` "w4a16": bf16 rows; "w4a8": rows in 8 bits."""

    def __init__(self, in_features: int, out_features: int, mode: str = "w4a16", bias: bool = False,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        _check_mode(mode)
        if in_features % ops.FP4_GROUP:
            raise ValueError(f"in_features must be a multiple of {ops.FP4_GROUP}, got {in_features}")
        self.in_features, self.out_features, self.mode = in_features, out_features, mode
        tiles = -(-out_features // 16)
        self.register_buffer("qweight", torch.zeros((tiles, -(-in_features // 128), 1024), dtype=torch.uint8,
                                                    device=device))
        self.register_buffer("scales", torch.full((tiles, -(-in_features // 512), 256), 127, dtype=torch.uint8,
                                                  device=device))
        self.register_buffer("bias", torch.zeros((out_features,), dtype=torch.bfloat16, device=device) if bias else None)

    @classmethod
    def from_linear(cls, linear: nn.Linear, mode: str = "w4a16") -> Fp4Linear:
        """Quantizes `linear.weight` on its own (GPU) device."""
        check_fp4_supported(linear)
        mod = cls.from_quantized(*ops.quantize_weight_fp4(linear.weight.detach()), mode)
        if linear.bias is not None:
            mod.register_buffer("bias", linear.bias.detach().to(torch.bfloat16).clone())
        return mod

    @classmethod
    def from_quantized(cls, codes: torch.Tensor, scales: torch.Tensor, mode: str = "w4a16",
                       bias: torch.Tensor | None = None) -> Fp4Linear:
        """Wraps a weight that is quantized already: codes uint8 (N, K / 2), the lower k in the low half, and scales
        float8_e8m0fnu (N, K / 32), on the GPU."""
        weight = ops.pack_fp4(codes, scales)
        mod = cls(weight.k, weight.n, mode, bias is not None, "meta")
        mod.register_buffer("qweight", weight.codes)
        mod.register_buffer("scales", weight.scales.view(torch.uint8))
        if bias is not None:
            mod.register_buffer("bias", bias.to(weight.codes.device, torch.bfloat16))
        return mod

    def dequantized(self) -> torch.Tensor:
        """The weight's values, (N, K) fp32."""
        return ops.dequantize_fp4(*ops.unpack_fp4(ops.Fp4Weight(self.qweight, self.scales, self.out_features,
                                                                self.in_features)))

    def forward(self, x: torch.Tensor | QuantizedRows) -> torch.Tensor:
        group = self.__dict__.get("_qkv_group")
        if group is not None:
            y = group.columns(self, x)
        else:
            y = _fp4_product(self.mode, x, self.qweight, self.scales, self.out_features, self.in_features)
        return y if self.bias is None else y + self.bias

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, mode={self.mode}, "
                f"bias={self.bias is not None}")


class Fp4QKVGroup(QKVGroup):
    """`QKVGroup` over 4-bit weights: row tiles of codes and of scales stack alike."""

    def _product(self, x: torch.Tensor | QuantizedRows) -> torch.Tensor:
        return _fp4_product(self.mode, x, self.qweight, self.scales, self.n, self.members[0].in_features)

    def _members_are_views(self) -> bool:
        for mod in self.members:
            tile = self.offsets[id(mod)][0] // 16
            for whole, part in ((self.qweight, mod._buffers["qweight"]), (self.scales, mod._buffers["scales"])):
                if (part.device != whole.device or part.dtype != whole.dtype
                        or part.data_ptr() != whole.data_ptr() + tile * whole.stride(0)):
                    return False
        return True

    def _restack(self) -> None:
        self._stack()

    def _stack(self) -> None:
        """Makes the members' buffers views of their stack."""
        self.qweight = torch.cat([m._buffers["qweight"] for m in self.members])
        self.scales = torch.cat([m._buffers["scales"] for m in self.members])
        for m in self.members:
            a, b = (v // 16 for v in self.offsets[id(m)])
            m._buffers["qweight"], m._buffers["scales"] = self.qweight[a:b], self.scales[a:b]


def group_qkv_fp4(attn: nn.Module) -> Fp4QKVGroup | None:
    """`group_qkv` for Fp4Linear projections."""
    def make(mods: list[Fp4Linear]) -> Fp4QKVGroup:
        group = Fp4QKVGroup(mods[0].qweight, mods[0].scales, mods[0].mode, mods)
        group._stack()
        return group

    return group_qkv_as(attn, Fp4Linear, make)


class Fp4GateUp(nn.Module):
    """h = silu(x · Gᵀ) * (x · Uᵀ), x (..., K) → h (..., I) bf16, gate and up weights in 4 bits: one kernel, rounded
    once."""

    def __init__(self, weight: ops.Fp4Weight, mode: str = "w4a16") -> None:
        super().__init__()
        _check_mode(mode)
        self.in_features, self.intermediate_size, self.mode = weight.k, weight.n, mode
        self.register_buffer("qweight", weight.codes)
        self.register_buffer("scales", weight.scales.view(torch.uint8))

    @classmethod
    def from_linears(cls, gate: nn.Linear, up: nn.Linear, mode: str = "w4a16") -> Fp4GateUp:
        """Quantizes the bias-free `gate` and `up` projections."""
        for lin in (gate, up):
            check_fp4_supported(lin)
            if lin.bias is not None:
                raise RuntimeError("the fused gate/up kernel takes bias-free projections")
        if gate.weight.shape != up.weight.shape:
            raise RuntimeError(f"gate and up shapes differ: {tuple(gate.weight.shape)} vs {tuple(up.weight.shape)}")
        halves = [ops.quantize_weight_fp4(lin.weight.detach()) for lin in (gate, up)]
        codes = torch.cat([c for c, _ in halves])
        scales = torch.cat([s.view(torch.uint8) for _, s in halves]).view(torch.float8_e8m0fnu)
        return cls(ops.pack_fp4(codes, scales, glu=True), mode)

    def dequantized(self) -> torch.Tensor:
        """The stacked [gate; up] weight's values, (2 I, K) fp32."""
        return ops.dequantize_fp4(*ops.unpack_fp4(ops.Fp4Weight(self.qweight, self.scales, self.intermediate_size,
                                                                self.in_features)))

    def forward(self, x: torch.Tensor | QuantizedRows) -> torch.Tensor:
        x = _fp8_input(self.mode, x)
        weight = ops.Fp4Weight(self.qweight, self.scales, self.intermediate_size, self.in_features)
        return ops.w4a8_glu(x, weight) if self.mode == "w4a8" else ops.w4a16_glu(x, weight)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, intermediate_size={self.intermediate_size}, mode={self.mode}"


class Fp4GluMLP(nn.Module):
    """Drop-in for `LlamaMLP` (modeling_llama.py:163-176): forward(x) = down_proj(gate_up(x))."""

    def __init__(self, gate_up: Fp4GateUp, down_proj: Fp4Linear) -> None:
        super().__init__()
        self.gate_up = gate_up
        self.down_proj = down_proj

    @classmethod
    def from_mlp(cls, mlp: nn.Module, mode: str = "w4a16") -> Fp4GluMLP:
        """Quantizes a `LlamaMLP` (gate_proj, up_proj, down_proj, SiLU act_fn, no bias on gate and up)."""
        if not _is_silu(mlp.act_fn):
            raise RuntimeError(f"the fused gate/up kernel applies SiLU, the MLP uses {type(mlp.act_fn).__name__}")
        return cls(Fp4GateUp.from_linears(mlp.gate_proj, mlp.up_proj, mode), Fp4Linear.from_linear(mlp.down_proj, mode))

    def forward(self, x: torch.Tensor | QuantizedRows) -> torch.Tensor:
        return self.down_proj(self.gate_up(x))


class Fp8RMSNorm(nn.Module):
    """Drop-in for a decoder layer's norms in the mode "w4a8": the norm and the rounding of its rows to 8 bits, which
    each of its consumers would repeat, run as one kernel. The bf16 weight stays a Parameter."""

    def __init__(self, norm: nn.Module) -> None:
        super().__init__()
        self.weight = norm.weight
        self.variance_epsilon = norm.variance_epsilon

    def forward(self, x: torch.Tensor) -> QuantizedRows:
        _, rows = ops.add_rmsnorm_fp8(x, None, self.weight, self.variance_epsilon)
        return QuantizedRows(rows.codes, rows.scales, x.shape, x.dtype)

    def extra_repr(self) -> str:
        return f"{tuple(self.weight.shape)}, eps={self.variance_epsilon}, quantize=e4m3 by 32"
