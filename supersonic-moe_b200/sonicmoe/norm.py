"""Root-mean-square norm in front of the layer: the residual's addition, the norm, and the 8-bit payload that the experts take, in one
pass over the rows.  Not part of the reference signature, whose layer begins behind it.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import host as _host
from .functional import _after_accumulate, _base_of, _grad_target


class NormQuantized(NamedTuple):
    """What `rms_norm_quantized` returns: e4m3 payload and scales of the rows, the rows in bf16 (or None), and the sum x + residual
    (or None)."""
    payload: torch.Tensor
    scales: torch.Tensor
    y: torch.Tensor | None
    h: torch.Tensor | None


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
        main_grad = None
        if need_w:
            main_grad, base = _grad_target(ctx.weight, ctx.weight.shape)
        if dy is None:                                   # only the sum was used
            if main_grad is not None:
                _after_accumulate(base)
            return (dh.to(tx) if need_x and dh is not None else None, torch.zeros_like(w) if need_w and main_grad is None else None,
                    dh if need_r else None, None, None)
        apart = tr is not None and tr != tx
        dx, dres, dw = ops.rms_norm_bwd(dy.contiguous(), h, w, r, None if dh is None else dh.contiguous(),
                                        need_x or (need_r and not apart), need_r and apart, need_w, main_grad)
        if main_grad is not None:
            _after_accumulate(base)
        return dx if need_x else None, dw, (dres if apart else dx) if need_r else None, None, None


def _call(x, weight, residual, eps, scales, with_output):
    """payload, scales, y, h"""
    kind = ops.NORM_SCALES[scales]
    grad = torch.is_grad_enabled()
    if ops._recorder is None and not (grad and weight.requires_grad and getattr(_base_of(weight), "main_grad", None) is not None):
        return _host.norm_call(x, weight, residual, eps, kind, with_output)
    rows, w, res = _host.norm_checked(x, weight, residual, eps, kind)
    if grad and (rows.requires_grad or w.requires_grad or (res is not None and res.requires_grad)):
        if scales and not with_output:
            raise ValueError("rms_norm_quantized: no gradient flows through the payload; with_output=True gives the rows it flows through")
        y, h, q, s = _RmsNorm.apply(rows, w, res, eps, scales)
    else:
        y, h, q, s, _ = ops.rms_norm(rows, w, res, eps, scales, with_output)
    return _host.norm_in_shape(x, q, s, y, h)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *, eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last dimension, h = x, or x + residual; returns y, with a residual (y, h).

    x bf16 or f32 [..., H], 1 <= H <= 16384, rows any distance apart; weight bf16 or f32 [H]; residual of x's shape and of x's type or
    f32.  y is of x's type, h of the residual's: it is rounded to that type, and the norm is that of the rounded sum, so that the next
    layer and the backward pass see the same rows.  Mean and root are f64; bf16 results are those of 64 bits (but where h / sqrt(...) lies
    below f32's normal range, 2^-126), and what lies within 2^-50 of the middle between two bf16 goes to the even one.
    eps is 0 or at least 1e-90.

    Differentiable in x, weight and residual (the gradient of h included); a weight's gradient goes to the parameter's f32 `main_grad`
    where it has one.  Gradients cannot be differentiated again, and there are no forward-mode derivatives."""
    _, _, y, h = _call(x, weight, residual, eps, None, True)
    return y if residual is None else (y, h)


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
    return NormQuantized._make(_call(x, weight, residual, eps, scales, with_output))
