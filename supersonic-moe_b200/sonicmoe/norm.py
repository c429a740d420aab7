"""Root-mean-square norm in front of the layer: the residual's addition, the norm, and the 8-bit payload that the experts take, in one
pass over the rows.  Not part of the reference signature, whose layer begins behind it.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _host, ops
from .functional import _after_accumulate, _base_of, _grad_target

_TYPES = (torch.bfloat16, torch.float32)


class NormQuantized(NamedTuple):
    """What `rms_norm_quantized` returns: e4m3 payload and scales of the rows, the rows in bf16 (or None), and the sum x + residual
    (or None)."""
    payload: torch.Tensor
    scales: torch.Tensor
    y: torch.Tensor | None
    h: torch.Tensor | None


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., H] as [rows, H] whose values lie side by side; the rows may be any distance apart."""
    t = t if t.ndim == 2 else t.reshape(-1, t.shape[-1])
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


class _RmsNorm(torch.autograd.Function):
    """x, residual [rows,H] (residual or None), weight [H] -> y, h, payload, scales, each None where there is none: for a weight that
    accumulates into its `main_grad`.  (Others have their node in csrc/host_torch.cpp.)"""

    @staticmethod
    def forward(ctx, x, weight, residual, eps, scales):
        y, h, q, s, r = ops.rms_norm(x, weight, residual, eps, scales, True, True)
        ctx.save_for_backward(x if h is None else h, weight, r)
        ctx.weight, ctx.types = weight, (x.dtype, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        if q is not None:
            ctx.mark_non_differentiable(q, s)
        return y, h, q, s

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh, _dq, _ds):
        h, w, r = ctx.saved_tensors
        tx, tr = ctx.types
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        if dy is None:                                   # only the sum was used
            return (dh.to(tx) if need_x and dh is not None else None, torch.zeros_like(w) if need_w else None,
                    dh if need_r else None, None, None)
        main_grad = None
        if need_w:
            main_grad, base = _grad_target(ctx.weight, ctx.weight.shape)
        apart = tr is not None and tr != tx
        dx, dres, dw = ops.rms_norm_bwd(dy.contiguous(), h, w, r, None if dh is None else dh.contiguous(),
                                        need_x or (need_r and not apart), need_r and apart, need_w, main_grad)
        if main_grad is not None:
            _after_accumulate(base)
        return dx if need_x else None, dw, (dres if apart else dx) if need_r else None, None, None


def _checked(x, weight, residual, eps, what, types):
    H = x.shape[-1] if x.ndim else 0
    if x.dtype not in types:
        raise ValueError(f"{what}: x is {' or '.join(str(t) for t in types)}, got {x.dtype}")
    if not 1 <= H <= ops.NORM_MAX_H:
        raise ValueError(f"{what}: rows have 1 to {ops.NORM_MAX_H} values, got {tuple(x.shape)}")
    if weight.dtype not in _TYPES or weight.shape != (H,):
        raise ValueError(f"{what}: the weight is bf16 or f32 [{H}], got {weight.dtype} {tuple(weight.shape)}")
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f"{what}: the residual is {x.dtype} or f32 {tuple(x.shape)}, got {residual.dtype} {tuple(residual.shape)}")
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"{what}: eps={eps}")
    return weight if weight.is_contiguous() else weight.contiguous()


def _needs_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _differentiable(rows, w, res, eps, scales):
    """y, h, payload, scales."""
    if ops._recorder is not None or (w.requires_grad and getattr(_base_of(w), "main_grad", None) is not None):
        return _RmsNorm.apply(rows, w, res, eps, scales)
    out = _host.rms_norm_grad(rows, w, res, eps, ops.NORM_SCALES[scales])
    h = out[1] if res is not None else None
    return (out[0], h, out[-2], out[-1]) if scales else (out[0], h, None, None)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension, h = x, or x + residual; returns y, with a residual (y, h).

    x bf16 or f32 [..., H], 1 <= H <= 16384, rows any distance apart; weight bf16 or f32 [H]; residual of x's shape and of x's type or
    f32.  y is of x's type, h of the residual's: it is rounded to that type, and the norm is that of the rounded sum, so that the next
    layer and the backward pass see the same rows.  Mean and root are f64; bf16 results are those of 64 bits.

    Differentiable in x, weight and residual (the gradient of h included); a weight's gradient goes to the parameter's f32 `main_grad`
    where it has one.  Gradients cannot be differentiated again."""
    w = _checked(x, weight, residual, eps, "rms_norm", _TYPES)
    rows, res = _rows(x), None if residual is None else _rows(residual)
    if _needs_grad(x, weight, residual):
        y, h = _differentiable(rows, w, res, eps, None)[:2]
    else:
        y, h = ops.rms_norm(rows, w, res, eps)[:2]
    y = y if x.ndim == 2 else y.view(x.shape)
    return y if residual is None else (y, h if x.ndim == 2 else h.view(x.shape))


def rms_norm_quantized(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6,
                       scales: str = "mx", with_output: bool = False) -> NormQuantized:
    """`rms_norm` of bf16 rows and, from the same pass, what a row quantiser makes of its y: (payload, scales, y, h).

    scales "mx": payload e4m3 [..., H], scales u8 [..., H/32] (ue8m0 per 1x32, H % 32 == 0), as `run_sonic_moe` takes them with
    `fp8_scale`; "block128": scales f32 [..., ceil(H/128)], as `quantize_rows_block128` makes them (H % 8 == 0; where H is no multiple of
    16 the payload is a view whose rows start on 16-byte boundaries).  Bit for bit the quantiser's output on y.  y is None without
    `with_output`, h without a residual.

    No gradient flows through 8 bits: a call whose inputs need one has to ask for y, and hands it to the experts beside the payload
    (`run_sonic_moe(payload, ..., fp8_scale=scales, grad_holder=y)`), so that theirs reaches the norm as y's gradient, along with the
    router's."""
    if scales not in ("mx", "block128"):
        raise ValueError(f"rms_norm_quantized: scales={scales!r}: 'mx' or 'block128'")
    w = _checked(x, weight, residual, eps, "rms_norm_quantized", (torch.bfloat16,))
    H, unit = x.shape[-1], 32 if scales == "mx" else 8
    if H % unit:
        raise ValueError(f"rms_norm_quantized: {H} columns are no multiple of {unit} (scales={scales!r})")
    rows, res = _rows(x), None if residual is None else _rows(residual)
    if _needs_grad(x, weight, residual):
        if not with_output:
            raise ValueError("rms_norm_quantized: no gradient flows through the payload; with_output=True gives the rows it flows through")
        y, h, q, s = _differentiable(rows, w, res, eps, scales)
    else:
        y, h, q, s, _ = ops.rms_norm(rows, w, res, eps, scales, with_output)
    if x.ndim != 2:
        lead = x.shape[:-1]
        q, s = q.unflatten(0, lead) if lead else q[0], s.unflatten(0, lead) if lead else s[0]
        y, h = (t if t is None else t.view(x.shape) for t in (y, h))
    return NormQuantized(q, s, y, h)
