"""Fused element-wise companions of the LoRA'd linears inside a DiT block, with autograd:

    modulated_layer_norm(x, shift, scale) = layer_norm(x) * (1 + scale) + shift
    gated_residual(x, gate, y)            = x + gate * y
    swiglu(gate, up)                      = silu(gate) * up           (mmdit.rs:695-708)
    sigmoid_gate(x, gate)                 = x * sigmoid(gate)         (mmdit.rs:659-664)
    zrmsnorm(x, scale)                    = x / sqrt(mean(x^2) + 1e-5) * (scale + 1)   (mmdit.rs:282-330)
    modulated_zrmsnorm(x, w, shift, scale) = zrmsnorm(x, w) * (1 + scale) + shift
    gated_residual_norm(x, gate, y, ..)   = r = a x + gate * post(y) and the modulated norm of r, in one pass

the pattern of crates/loractl-core/src/mmdit.rs:857-869 (`(prescale + 1) * prenorm(x) + preshift`,
`x + pregate * attn(..)`, ...).  `x`, `y` are `[b, tokens, h]`; `shift`, `scale`, `gate` are
`[b, 1, h]` (or `[b, h]`) and broadcast over the tokens of their sample.  Each op is one kernel
forward; the backward is one pass for the token-shaped gradient plus a fixed-order two-stage sum
over tokens for the modulation gradients (deterministic, as block-checkpoint recompute needs).
CUDA tensors only (f32 or bf16): like every other op of this package there is no CPU path.
"""
from __future__ import annotations

import functools
import struct
from typing import Dict, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from .quant import _dtype_code, _on_device, _raw_stream, _require_cuda, _stream_ptr

LN_EPS = 1e-5  # torch.nn.functional.layer_norm's default, which the harness block used before

_WS: Dict[Tuple[torch.device, int], torch.Tensor] = {}


def _workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    key = (device, torch.cuda.current_stream(device).cuda_stream)
    ws = _WS.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _WS[key] = ws
    return ws


def _dims(x: torch.Tensor) -> Tuple[int, int, int]:
    if x.dim() != 3:
        raise ValueError(f"expected [b, tokens, h], got {list(x.shape)}")
    return x.shape[0], x.shape[1], x.shape[2]


def _mod(v: torch.Tensor, b: int, h: int, like: torch.Tensor, name: str) -> torch.Tensor:
    if v.numel() != b * h:
        raise ValueError(f"{name} must hold [b = {b}, h = {h}] values, got {list(v.shape)}")
    return v.reshape(b, h).to(like.dtype).contiguous()


class _ModulatedLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, shift, scale):
        _require_cuda(x, "x")
        b, t, h = _dims(x)
        xc = x.contiguous()
        sh, sc = _mod(shift, b, h, xc, "shift"), _mod(scale, b, h, xc, "scale")
        y = torch.empty_like(xc)
        mean = torch.empty(b * t, dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
        with torch.cuda.device(x.device):
            L.check(L.lib().lq_ln_modulate_fwd(xc.data_ptr(), sh.data_ptr(), sc.data_ptr(), _dtype_code(xc), b, t, h,
                                               LN_EPS, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                               _stream_ptr(x.device)))
        ctx.save_for_backward(xc, sc, mean, rstd)
        ctx.shapes = (shift.shape, scale.shape, shift.dtype, scale.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        xc, sc, mean, rstd = ctx.saved_tensors
        b, t, h = _dims(xc)
        dyc = dy.contiguous()
        dx = torch.empty_like(xc)
        dshift = torch.empty((b, h), dtype=torch.float32, device=xc.device)
        dscale = torch.empty_like(dshift)
        with torch.cuda.device(xc.device):
            n = L.lib().lq_block_ops_workspace_bytes(b, t, h)
            ws = _workspace(xc.device, n)
            L.check(L.lib().lq_ln_modulate_bwd(dyc.data_ptr(), xc.data_ptr(), sc.data_ptr(), mean.data_ptr(),
                                               rstd.data_ptr(), _dtype_code(xc), b, t, h, dx.data_ptr(),
                                               dshift.data_ptr(), dscale.data_ptr(), ws.data_ptr(), ws.numel(),
                                               _stream_ptr(xc.device)))
        shs, scs, shd, scd = ctx.shapes
        return dx, dshift.to(shd).reshape(shs), dscale.to(scd).reshape(scs)


class _GatedResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, y):
        _require_cuda(y, "y")
        b, t, h = _dims(y)
        yc = y.contiguous()
        xc = x.to(yc.dtype).contiguous()
        g = _mod(gate, b, h, yc, "gate")
        out = torch.empty_like(yc)
        with torch.cuda.device(y.device):
            L.check(L.lib().lq_gate_residual_fwd(xc.data_ptr(), g.data_ptr(), yc.data_ptr(), _dtype_code(yc), b, t, h,
                                                 out.data_ptr(), _stream_ptr(y.device)))
        ctx.save_for_backward(g, yc)
        ctx.meta = (gate.shape, gate.dtype, x.dtype)
        return out

    @staticmethod
    def backward(ctx, dout):
        g, yc = ctx.saved_tensors
        b, t, h = _dims(yc)
        dc = dout.contiguous()
        dy = torch.empty_like(yc)
        dgate = torch.empty((b, h), dtype=torch.float32, device=yc.device)
        with torch.cuda.device(yc.device):
            n = L.lib().lq_block_ops_workspace_bytes(b, t, h)
            ws = _workspace(yc.device, n)
            L.check(L.lib().lq_gate_residual_bwd(dc.data_ptr(), g.data_ptr(), yc.data_ptr(), _dtype_code(yc), b, t, h,
                                                 dy.data_ptr(), dgate.data_ptr(), ws.data_ptr(), ws.numel(),
                                                 _stream_ptr(yc.device)))
        gs, gd, xd = ctx.meta
        return dc.to(xd), dgate.to(gd).reshape(gs), dy


def modulated_layer_norm(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """`layer_norm(x, (h,)) * (1 + scale) + shift`, one kernel."""
    return _ModulatedLayerNorm.apply(x, shift, scale)


def gated_residual(x: torch.Tensor, gate: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """`x + gate * y`, one kernel."""
    return _GatedResidual.apply(x, gate, y)


class _PairAct(torch.autograd.Function):
    """Element-wise map of two same-shaped tensors with both input gradients from one backward pass."""

    @staticmethod
    def forward(ctx, a, b, kind):
        _require_cuda(a, "input")
        if a.shape != b.shape or a.dtype != b.dtype:
            raise ValueError(f"operands must agree in shape and dtype, got {list(a.shape)} {a.dtype} / {list(b.shape)} {b.dtype}")
        ac, bc = a.contiguous(), b.contiguous()
        out = torch.empty_like(ac)
        fn = L.lib().lq_swiglu_fwd if kind == "swiglu" else L.lib().lq_sigmoid_gate_fwd
        with torch.cuda.device(a.device):
            L.check(fn(ac.data_ptr(), bc.data_ptr(), _dtype_code(ac), ac.numel(), out.data_ptr(), _stream_ptr(a.device)))
        ctx.save_for_backward(ac, bc)
        ctx.kind = kind
        return out

    @staticmethod
    def backward(ctx, dout):
        ac, bc = ctx.saved_tensors
        dc = dout.to(ac.dtype).contiguous()
        da, db = torch.empty_like(ac), torch.empty_like(bc)
        fn = L.lib().lq_swiglu_bwd if ctx.kind == "swiglu" else L.lib().lq_sigmoid_gate_bwd
        with torch.cuda.device(ac.device):
            L.check(fn(dc.data_ptr(), ac.data_ptr(), bc.data_ptr(), _dtype_code(ac), ac.numel(), da.data_ptr(),
                       db.data_ptr(), _stream_ptr(ac.device)))
        return da, db, None


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """`silu(gate) * up`, one kernel each way."""
    return _PairAct.apply(gate, up, "swiglu")


def sigmoid_gate(x: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
    """`x * sigmoid(gate)`, one kernel each way."""
    return _PairAct.apply(x, gate, "sigmoid_gate")


ZRMS_EPS = 1e-5  # crates/loractl-core/src/mmdit.rs:282-330


class _ZRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, scale):
        _require_cuda(x, "x")
        h = x.shape[-1]
        if scale.numel() != h:
            raise ValueError(f"scale must hold {h} values, got {list(scale.shape)}")
        xc = x.contiguous()
        sc = scale.detach().to(torch.float32).contiguous()
        rows = xc.numel() // h
        y = torch.empty_like(xc)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        with torch.cuda.device(x.device):
            L.check(L.lib().lq_zrmsnorm_fwd(xc.data_ptr(), sc.data_ptr(), _dtype_code(xc), rows, h, ZRMS_EPS, y.data_ptr(),
                                            rstd.data_ptr(), _stream_ptr(x.device)))
        ctx.save_for_backward(xc, sc, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        xc, sc, rstd = ctx.saved_tensors
        h = xc.shape[-1]
        dc = dy.to(xc.dtype).contiguous()
        dx = torch.empty_like(xc)
        with torch.cuda.device(xc.device):
            L.check(L.lib().lq_zrmsnorm_bwd(dc.data_ptr(), xc.data_ptr(), sc.data_ptr(), rstd.data_ptr(), _dtype_code(xc),
                                            xc.numel() // h, h, dx.data_ptr(), _stream_ptr(xc.device)))
        return dx, None


def zrmsnorm(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """ZRmsNorm over the last axis with a frozen `scale` (no gradient flows to it), one kernel each way."""
    return _ZRmsNorm.apply(x, scale)


# ---- the seam between two sub-blocks --------------------------------------------------------------

# `lq_residual_norm_args` and `lq_residual_norm_grads` as one pack each: setting thirty ctypes fields takes longer
# than the kernel of a short call
_ARGS = struct.Struct("@12P10q3i2f0P")
_GRADS = struct.Struct("@2P4q7P")


@functools.lru_cache(maxsize=256)
def _residual_norm_ws(index: int, b: int, t: int, h: int) -> int:
    return L.lib().lq_residual_norm_workspace_bytes(b, t, h)


def _rows(v: torch.Tensor) -> torch.Tensor:
    """`v` itself when its rows are contiguous (any sample and token stride), a copy otherwise."""
    return v if v.stride(-1) == 1 or v.shape[-1] == 1 else v.contiguous()


def _vector(v: torch.Tensor, b: int, h: int, dtype: torch.dtype, name: str) -> torch.Tensor:
    """A modulation vector as a `[b, h]` view (a copy where its type differs or its rows are not contiguous)."""
    shape = v.shape
    if shape[-1] != h or shape[0] != b or v.numel() != b * h:
        raise ValueError(f"{name} must be [b = {b}, h = {h}] or [b, 1, h], got {list(shape)}")
    if v.dtype != dtype:
        v = v.to(dtype)
    if len(shape) != 2:
        v = v.reshape(b, h)
    return v if v.stride(1) == 1 or h == 1 else v.contiguous()


def _norm_weight(w: Optional[torch.Tensor], h: int, name: str) -> Optional[torch.Tensor]:
    if w is None:
        return None
    if w.numel() != h:
        raise ValueError(f"{name} must hold {h} values, got {list(w.shape)}")
    if w.dtype != torch.float32 or w.dim() != 1:
        w = w.to(torch.float32).reshape(h)
    return w if w.stride(0) == 1 else w.contiguous()


def _residual_norm(x, gate, y, shift, scale, weight, post_weight, layer, alpha, eps, want_stats):
    """The checks and the forward launch; returns (outputs, what the backward needs)."""
    _require_cuda(x, "x")
    b, t, h = _dims(x)
    dtype, device = _dtype_code(x), x.device
    if y is not None and (y.shape != x.shape or y.dtype != x.dtype):
        raise ValueError(f"x and y must agree in shape and dtype, got {list(x.shape)} {x.dtype} / {list(y.shape)} {y.dtype}")
    index = x.get_device()
    for name, v in (("gate", gate), ("y", y), ("shift", shift), ("scale", scale), ("weight", weight), ("post_weight", post_weight)):
        if v is not None and v.get_device() != index:
            raise RuntimeError(f"{name} is on {v.device}, x on {device}")
    # one type for the modulation vectors: theirs when they agree on f32 or bf16, else f32
    kinds = {v.dtype for v in (gate, shift, scale) if v is not None}
    if not kinds <= {torch.float32, torch.bfloat16}:
        raise TypeError(f"unsupported dtype of gate, shift or scale {sorted(map(str, kinds))}: f32 or bf16")
    mod_dtype = shift.dtype if len(kinds) == 1 else torch.float32
    gate = None if y is None else _vector(gate, b, h, mod_dtype, "gate")
    shift, scale = _vector(shift, b, h, mod_dtype, "shift"), _vector(scale, b, h, mod_dtype, "scale")
    w, pw = _norm_weight(weight, h, "weight"), _norm_weight(post_weight, h, "post_weight")
    x = _rows(x)
    z = torch.empty((b, t, h), dtype=x.dtype, device=device)
    r, yp, ys, gp, gs, rp = None, 0, (0, 0, 0), 0, 0, 0
    if y is not None:
        y = _rows(y)
        r = torch.empty_like(z)
        yp, ys, gp, gs, rp = y.data_ptr(), y.stride(), gate.data_ptr(), gate.stride(0), r.data_ptr()
    stats, sp = None, (0, 0, 0)
    if want_stats:
        stats = torch.empty((3, b * t), dtype=torch.float32, device=device)
        p = stats.data_ptr()
        sp = (p, p + 4 * b * t, p + 8 * b * t)
    xs = x.stride()
    args = _ARGS.pack(x.data_ptr(), yp, gp, shift.data_ptr(), scale.data_ptr(), 0 if w is None else w.data_ptr(),
                      0 if pw is None else pw.data_ptr(), rp, z.data_ptr(), *sp, xs[0], xs[1], ys[0], ys[1], gs, shift.stride(0),
                      scale.stride(0), b, t, h, dtype, mod_dtype == torch.float32, layer, alpha, eps)
    with _on_device(index):
        L.check(L.lib().lq_residual_norm_fwd(args, _raw_stream(index)))
    return (z,) if r is None else (r, z), (args, mod_dtype, (x, y, gate, shift, scale, w, pw, stats))


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        outs, (ctx.args, ctx.mod_dtype, saved) = _residual_norm(*inputs, True)
        # the addresses in `args` are those of the saved tensors; r and z among them are not read by the backward
        ctx.save_for_backward(*saved)
        ctx.like = [None if v is None else (v.shape, v.dtype) for v in (inputs[1], *inputs[3:7])]
        ctx.set_materialize_grads(False)
        return outs if len(outs) == 2 else outs[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, *douts):
        dr, dz = douts if len(douts) == 2 else (None, douts[0])
        if dr is None and dz is None:
            return (None,) * 10
        x = ctx.saved_tensors[0]  # the others only have to live
        b, t, h = x.shape
        dev, index, need = x.device, x.get_device(), ctx.needs_input_grad
        dx = torch.empty((b, t, h), dtype=x.dtype, device=dev) if need[0] else None
        dy = torch.empty((b, t, h), dtype=x.dtype, device=dev) if need[2] else None
        wanted = (need[1], need[3], need[4], need[5], need[6])
        grads = [None] * 5
        if any(wanted[:3]):  # one buffer for the three: a view each
            for i, v in enumerate(torch.empty((3, b, h), dtype=ctx.mod_dtype, device=dev).unbind(0)):
                grads[i] = v if wanted[i] else None
        if any(wanted[3:]):
            for i, v in enumerate(torch.empty((2, h), dtype=torch.float32, device=dev).unbind(0), 3):
                grads[i] = v if wanted[i] else None
        rp, rs, zp, zs = 0, (0, 0), 0, (0, 0)
        if dr is not None:
            dr = _rows(dr)
            rp, rs = dr.data_ptr(), dr.stride()
        if dz is not None:
            dz = _rows(dz)
            zp, zs = dz.data_ptr(), dz.stride()
        at = [0 if v is None else v.data_ptr() for v in (dx, dy, *grads)]
        g = _GRADS.pack(rp, zp, rs[0], rs[1], zs[0], zs[1], *at)
        with _on_device(index):
            ws, nbytes = None, 0
            if any(wanted):
                # of this call alone: from the pool of the current stream, or of the graph being captured
                nbytes = _residual_norm_ws(index, b, t, h)
                ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            L.check(L.lib().lq_residual_norm_bwd(ctx.args, g, None if ws is None else ws.data_ptr(), nbytes, _raw_stream(index)))
        for i, like in enumerate(ctx.like):
            if grads[i] is not None:
                v = grads[i] if grads[i].dtype == like[1] else grads[i].to(like[1])
                grads[i] = v if v.shape == like[0] else v.view(like[0])
        return dx, grads[0], dy, grads[1], grads[2], grads[3], grads[4], None, None, None


def _apply_residual_norm(*inputs):
    if torch.is_grad_enabled() and any(v is not None and v.requires_grad for v in inputs[:7]):
        return _ResidualNorm.apply(*inputs)
    outs, _ = _residual_norm(*inputs, False)
    return outs if len(outs) == 2 else outs[0]


def modulated_zrmsnorm(x: torch.Tensor, weight: Optional[torch.Tensor], shift: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """`zrmsnorm(x, weight) * (1 + scale) + shift` (mmdit.rs:857-862 before a sub-block), one kernel each way; `weight`
    `[h]` or None.  Gradients flow to every argument that asks for one, the norm's weight among them."""
    return _apply_residual_norm(x, None, None, shift, scale, weight, None, False, 1.0, ZRMS_EPS)


def gated_residual_norm(x: torch.Tensor, gate: torch.Tensor, y: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, *,
                        norm: str = "zrms", weight: Optional[torch.Tensor] = None,
                        post_weight: Optional[torch.Tensor] = None, residual_scale: float = 1.0
                        ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The end of one sub-block and the start of the next in one pass; returns `(r, z)`:

        r = residual_scale * x + gate * y          (y * rsqrt(mean(y^2) + eps) * (1 + post_weight) with a post_weight)
        z = norm(r) * (1 + weight) * (1 + scale) + shift

    `x`, `y`: `[b, tokens, h]`, f32 or bf16 alike, rows contiguous, samples and tokens at any stride; `gate`, `shift`,
    `scale`: `[b, 1, h]` or `[b, h]` (slices of one modulation tensor are read in place; expand over `b` to share a
    vector); `weight`, `post_weight`: `[h]` or None; h <= 16384.  `norm`: "zrms" (mmdit.rs:282-330) or "layer".
    Arithmetic is f32, `z` comes from the unrounded `r`, each output is rounded once; one kernel forward, one plus a
    fixed-order sum over tokens backward, gradients to every tensor argument that asks for one."""
    if norm not in ("zrms", "layer"):
        raise ValueError(f"norm must be zrms or layer, got {norm!r}")
    eps = ZRMS_EPS if norm == "zrms" else LN_EPS
    return _apply_residual_norm(x, gate, y, shift, scale, weight, post_weight, norm == "layer", float(residual_scale), eps)
