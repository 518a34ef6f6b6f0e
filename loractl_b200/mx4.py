"""Microscaled 4-bit floating point (MXFP4) as a frozen base: quantisation, the product of two microscaled tensors and
a linear layer on them — a second 4-bit format beside `quant.py`'s int4 (crates/loractl-core/src/quant.rs:52-82).

Elements are e2m1 floats under one power-of-two scale per 32 along a row.  The tensor cores multiply the format as it
is stored, so a product dequantises nothing; in exchange activations are quantised too, block by block, on the way in.
CUDA tensors only (f32 or bf16): there is no CPU path.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from .quant import _dtype_code, _on_device, _raw_stream, _require_cuda

MX4_BLOCK = 32
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


@functools.lru_cache(maxsize=512)
def _scale_bytes(rows: int, k: int) -> int:
    return L.lib().lq_mx4_scale_bytes(rows, k)


class Mx4Tensor:
    """A quantised `[rows, k]` tensor: `codes` (uint8 `[rows, k / 2]`, the even element in the low nibble) and `scales`
    (uint8, in the tiles that the tensor cores' copies read; `unpack` gives the logical view).  Immutable; never
    receives a gradient."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, k: int):
        need = _scale_bytes(rows, k)
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
        out = torch.empty((self.rows, self.k), dtype=dtype, device=self.device)
        code, index = _dtype_code(out), out.get_device()
        with _on_device(index):
            L.check(L.lib().lq_mx4_dequantize(self.codes.data_ptr(), self.scales.data_ptr(), self.rows, self.k, out.data_ptr(),
                                              code, _raw_stream(index)))
        return out

    def unpack(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Logical content: e2m1 codes (uint8 `[rows, k]`, sign in bit 3) and e8m0 scales (uint8 `[rows, k / 32]`)."""
        c = self.codes.view(self.rows, self.k // 2)
        codes = torch.stack((c & 15, c >> 4), dim=-1).reshape(self.rows, self.k)
        kt = 2 * -(-self.k // 256)
        tiles = self.scales.view(self.scales.numel() // (kt * 512), kt, 32, 4, 4)  # row tile, k tile, row % 32, row / 32, scale
        scales = tiles.permute(0, 3, 2, 1, 4).reshape(-1, kt * 4)[: self.rows, : self.k // 32]
        return codes, scales.contiguous()


@functools.lru_cache(maxsize=512)
def _linear_ws(n: int, k: int) -> int:
    return L.lib().lq_mx4_linear_workspace_bytes(n, k)


def _as_rows(x: torch.Tensor, k: int) -> torch.Tensor:
    """`x` as `[rows, k]` with contiguous rows that do not overlap."""
    x = x if x.dim() == 2 else x.reshape(-1, k)
    s0, s1 = x.stride()
    return x if s1 == 1 and (s0 >= k or x.shape[0] == 1) else x.contiguous()


def mx4_quantize(x: torch.Tensor) -> Mx4Tensor:
    """Quantises `x` `[..., k]` (f32 or bf16, k a multiple of 32) along its last axis, one kernel; leading axes become rows.
    A block of 32 gets the scale `2^(floor(log2(max |v|)) - 2)`, its elements round to nearest even and saturate at 6
    scales; a block that holds an Inf or a NaN stands for 32 NaNs."""
    _require_cuda(x, "x")
    dtype = _dtype_code(x)
    k = x.shape[-1] if x.dim() else 0
    if k == 0 or k % MX4_BLOCK:
        raise ValueError(f"the last axis must be a positive multiple of {MX4_BLOCK}, got {list(x.shape)}")
    x = _as_rows(x, k)
    rows, index = x.shape[0], x.get_device()
    q = Mx4Tensor.__new__(Mx4Tensor)
    q.rows, q.k = rows, k
    q.codes = torch.empty((rows, k // 2), dtype=torch.uint8, device=x.device)
    q.scales = torch.empty(_scale_bytes(rows, k), dtype=torch.uint8, device=x.device)
    with _on_device(index):
        L.check(L.lib().lq_mx4_quantize(x.data_ptr(), dtype, rows, k, x.stride(0), q.codes.data_ptr(), q.scales.data_ptr(),
                                        _raw_stream(index)))
    return q


def mx4_matmul_t(x: Mx4Tensor, w: Mx4Tensor, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """`dequant(x) . dequant(w)^T (+ bias)`, `[x.rows, w.rows]` in `dtype` (bf16 or f32), accumulated in f32 on the
    block-scaled tensor cores; `bias` f32 `[w.rows]`."""
    if not isinstance(x, Mx4Tensor) or not isinstance(w, Mx4Tensor):
        raise TypeError("mx4_matmul_t takes two microscaled tensors — see mx4_quantize")
    if x.k != w.k:
        raise ValueError(f"the block axes differ: {x.k} and {w.k}")
    if x.device != w.device:
        raise RuntimeError(f"x is on {x.device}, w on {w.device}")
    if bias is not None:
        if bias.numel() != w.rows or bias.device != w.device:
            raise ValueError(f"bias must hold {w.rows} values on {w.device}, got {list(bias.shape)} on {bias.device}")
        bias = bias.detach().to(torch.float32).contiguous()
    index = x.codes.get_device()
    y = torch.empty((x.rows, w.rows), dtype=dtype, device=x.device)
    code = _dtype_code(y)
    with _on_device(index):
        L.check(L.lib().lq_mx4_matmul(x.codes.data_ptr(), x.scales.data_ptr(), x.rows, w.codes.data_ptr(), w.scales.data_ptr(), w.rows,
                                      x.k, None if bias is None else bias.data_ptr(), y.data_ptr(), code, _raw_stream(index)))
    return y


def mx4_matmul_dx(dy: torch.Tensor, w: Mx4Tensor) -> torch.Tensor:
    """`dy [n, w.rows] . dequant(w)` in `dy`'s type: bf16 on the tensor cores (the weight is exact in bf16) or f32."""
    _require_cuda(dy, "dy")
    if dy.dim() != 2 or dy.shape[1] != w.rows:
        raise ValueError(f"dy must be [n, {w.rows}], got {list(dy.shape)}")
    index = dy.get_device()
    if index != w.codes.get_device():
        raise RuntimeError(f"dy is on {dy.device}, w on {w.device}")
    dtype = _dtype_code(dy)
    dy = dy.contiguous()
    if dy.data_ptr() % 16:
        dy = dy.clone()
    n = dy.shape[0]
    dx = torch.empty((n, w.k), dtype=dy.dtype, device=dy.device)
    lib = L.lib()
    with _on_device(index):
        ws = torch.empty(lib.lq_mx4_matmul_dx_workspace_bytes(n, w.rows, w.k, dtype), dtype=torch.uint8, device=dy.device)
        L.check(lib.lq_mx4_matmul_dx(dy.data_ptr(), dtype, n, w.codes.data_ptr(), w.scales.data_ptr(), w.rows, w.k, dx.data_ptr(),
                                     ws.data_ptr(), ws.numel(), _raw_stream(index)))
    return dx


def _linear(x: torch.Tensor, w: Mx4Tensor, bias: Optional[torch.Tensor]) -> torch.Tensor:
    """Quantisation and product of `x` `[n, k]`, one call."""
    _require_cuda(x, "x")
    dtype, index = _dtype_code(x), x.get_device()
    if index != w.codes.get_device():
        raise RuntimeError(f"x is on {x.device}, w on {w.device}")
    n, m, k = x.shape[0], w.rows, w.k
    x = _as_rows(x, k)
    y = torch.empty((n, m), dtype=x.dtype, device=x.device)
    with _on_device(index):
        nbytes = _linear_ws(n, k)  # of this call alone: from the pool of the current stream, or of the graph being captured
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        L.check(L.lib().lq_mx4_linear(x.data_ptr(), dtype, n, x.stride(0), w.codes.data_ptr(), w.scales.data_ptr(), m, k,
                                      None if bias is None else bias.data_ptr(), y.data_ptr(), ws.data_ptr(), nbytes, _raw_stream(index)))
    return y


class _Mx4Linear(torch.autograd.Function):
    """Forward `dequant(quant(x)) . dequant(w)^T + bias`; backward `dy . dequant(w)`, the quantisation of x taken as
    the identity.  The weight is state (quant.rs:217-219), never a graph parent."""

    @staticmethod
    def forward(ctx, x2, w, bias):
        ctx.w = w
        return _linear(x2, w, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return mx4_matmul_dx(dy, ctx.w), None, None


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
        if x.shape[-1] != self.d_in:
            raise ValueError(f"last dim {x.shape[-1]} != d_in {self.d_in}")
        x2 = x if x.dim() == 2 else x.reshape(-1, self.d_in)
        apply = _Mx4Linear.apply if x.requires_grad and torch.is_grad_enabled() else _linear
        y = apply(x2, self.weight, self.bias)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], self.d_out)
