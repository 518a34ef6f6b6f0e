"""Microscaled 4-bit floating point (MXFP4) as a frozen base: quantisation, the product of two microscaled tensors and
a linear layer on them — a second 4-bit format beside `quant.py`'s int4 (crates/loractl-core/src/quant.rs:52-82).

Elements are e2m1 floats under one power-of-two scale per 32 along a row.  The tensor cores multiply the format as it
is stored, so a product dequantises nothing; in exchange activations are quantised too, block by block, on the way in.
CUDA tensors only (f32 or bf16): there is no CPU path.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import nn

from . import _lib as L

MX4_BLOCK = 32


class Mx4Tensor:
    """A quantised `[rows, k]` tensor: `codes` (uint8 `[rows, k / 2]`, the even element in the low nibble) and `scales`
    (uint8, in the tiles that the tensor cores' copies read; `unpack` gives the logical view).  Immutable; never
    receives a gradient."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, k: int):
        need = L.lib().lq_mx4_scale_bytes(rows, k)
        for name, t, n in (("codes", codes, rows * k // 2), ("scales", scales, need)):
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != n:
                raise ValueError(f"{name} must be {n} contiguous bytes, got {list(t.shape)} {t.dtype}")
        if codes.device != scales.device:
            raise RuntimeError(f"codes are on {codes.device}, scales on {scales.device}")
        self.codes, self.scales, self.rows, self.k = codes, scales, rows, k

    @property
    def shape(self) -> Tuple[int, int]:
        return self.rows, self.k

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values it stands for, `[rows, k]`: exact in f32 and in bf16."""
        return L.ext().mx4_dequantize(self.codes, self.scales, self.rows, self.k, dtype)

    def unpack(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Logical content: e2m1 codes (uint8 `[rows, k]`, sign in bit 3) and e8m0 scales (uint8 `[rows, k / 32]`)."""
        c = self.codes.view(self.rows, self.k // 2)
        codes = torch.stack((c & 15, c >> 4), dim=-1).reshape(self.rows, self.k)
        kt = 2 * -(-self.k // 256)
        tiles = self.scales.view(self.scales.numel() // (kt * 512), kt, 32, 4, 4)  # row tile, k tile, row % 32, row / 32, scale
        scales = tiles.permute(0, 3, 2, 1, 4).reshape(-1, kt * 4)[: self.rows, : self.k // 32]
        return codes, scales.contiguous()


def mx4_quantize(x: torch.Tensor) -> Mx4Tensor:
    """Quantises `x` `[..., k]` (f32 or bf16, k a multiple of 32) along its last axis, one kernel; leading axes become rows.
    A block of 32 gets the scale `2^(floor(log2(max |v|)) - 2)`, its elements round to nearest even and saturate at 6
    scales; a block that holds an Inf or a NaN stands for 32 NaNs."""
    q = Mx4Tensor.__new__(Mx4Tensor)
    q.codes, q.scales = L.ext().mx4_quantize(x)
    q.rows, q.k = q.codes.shape[0], 2 * q.codes.shape[1]
    return q


def mx4_matmul_t(x: Mx4Tensor, w: Mx4Tensor, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """`dequant(x) . dequant(w)^T (+ bias)`, `[x.rows, w.rows]` in `dtype` (bf16 or f32), accumulated in f32 on the
    block-scaled tensor cores; `bias` f32 `[w.rows]`."""
    if not isinstance(x, Mx4Tensor) or not isinstance(w, Mx4Tensor):
        raise TypeError("mx4_matmul_t takes two microscaled tensors — see mx4_quantize")
    if x.k != w.k:
        raise ValueError(f"the block axes differ: {x.k} and {w.k}")
    return L.ext().mx4_matmul(x.codes, x.scales, x.rows, w.codes, w.scales, w.rows, w.k, bias, dtype)


def mx4_matmul_dx(dy: torch.Tensor, w: Mx4Tensor) -> torch.Tensor:
    """`dy [n, w.rows] . dequant(w)` in `dy`'s type: bf16 on the tensor cores (the weight is exact in bf16) or f32 (as three bf16
    terms of dy, exact but for what an element has below 2^-133)."""
    return L.ext().mx4_matmul_dx(dy, w.codes, w.scales, w.rows, w.k)


class Mx4Linear(nn.Module):
    """A frozen linear `[d_out, d_in]` in MXFP4: stands where `QuantLinear` does
    (crates/loractl-core/src/mmdit.rs:413-428).  x `[..., d_in]` is quantised on the way in; the output has x's type."""

    def __init__(self, weight: Mx4Tensor, bias: Optional[torch.Tensor] = None):
        super().__init__()
        if bias is not None and bias.numel() != weight.rows:
            raise ValueError(f"bias has {bias.numel()} elements, expected d_out = {weight.rows}")
        self.weight = weight
        self.d_out, self.d_in = weight.shape
        self.bias = None if bias is None else bias.detach().to(weight.device, torch.float32).contiguous()

    @staticmethod
    def from_linear(lin: nn.Linear) -> "Mx4Linear":
        return Mx4Linear(mx4_quantize(lin.weight), None if lin.bias is None else lin.bias)

    def dequantized_weight(self) -> torch.Tensor:
        """mmdit.rs:435-444 — diagnostics only."""
        return self.weight.dequantize()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """`dequant(quant(x)) . dequant(w)^T + bias`, quantisation and product in one call.  The gradient of x is
        `dy . dequant(w)`: the quantisation of x is taken as the identity, the weight is state (quant.rs:217-219)."""
        w = self.weight
        return L.ext().mx4_linear(x, w.codes, w.scales, w.rows, w.k, self.bias)

    def forward_adapted(self, x: torch.Tensor, delta) -> torch.Tensor:
        """`forward(x) + scaling * (x . lora_a) . lora_b` of a `LoraDelta` in one call, x in bf16 and d_out a multiple of 8: the
        adapter reads x itself, its factors rounded to bf16; the backward gives dx and both factors' gradients, into the
        flat gradient buffer where the factors live in one."""
        w, bucket = self.weight, delta.bucket_grads or (None, None)
        return L.ext().mx4_lora_linear(x, w.codes, w.scales, w.rows, w.k, self.bias, delta.lora_a, delta.lora_b, delta.scaling,
                                       delta.operand_mirror(), *bucket)
