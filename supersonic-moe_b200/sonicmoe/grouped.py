"""Products of bf16 rows grouped by expert, over segments that begin and end at any row: the experts' projections in the precision of
their weights, beside the 8-bit forms.  The signature is that of `block128_linear`; not part of the reference's.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import host as _host
from .functional import _after_accumulate, _base_of, _grad_target


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """[rows, n] that the copy engine can read as it lies: rows a multiple of 16 bytes apart and from a 16-byte boundary on."""
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (t.stride(0) >= t.shape[1] and t.stride(0) % 8 == 0)):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _weight16(w: torch.Tensor) -> torch.Tensor:
    w = w.detach().contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


class _GroupedLinear(torch.autograd.Function):
    """x [rows,K], weight bf16 [E,N,K] or [N,K] that accumulates into its `main_grad`.  (Others have their node in
    csrc/host_torch.cpp.)"""

    @staticmethod
    def forward(ctx, x, weight, efo, counts):
        w = _weight16(weight)
        w3 = w if w.ndim == 3 else w[None]
        y = ops.grouped_rows(x, w3, efo, counts)
        need_x, need_w = ctx.needs_input_grad[:2]
        # (the weight itself where it is read as it lies: autograd then sees a change in place between the passes)
        ctx.save_for_backward(x if need_w else None, (weight if w.data_ptr() == weight.data_ptr() else w) if need_x else None, efo, counts)
        ctx.weight, ctx.shape = weight if need_w else None, tuple(w3.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, efo, counts = ctx.saved_tensors
        dy = _rows16(dy)
        dx = dw = None
        if w is not None:
            dx = ops.grouped_rows(dy, w.detach().view(ctx.shape), efo, counts, True)
        if x is not None:
            main_grad, base = _grad_target(ctx.weight, ctx.weight.shape)
            dw = ops.grouped_wgrad(dy, x, efo, counts, ctx.shape[0], main_grad)
            if main_grad is not None:
                _after_accumulate(base)
            else:
                dw = dw.view(ctx.weight.shape)
        return dx, dw, None, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, efo: torch.Tensor | None = None,
                   counts: torch.Tensor | None = None) -> torch.Tensor:
    """y[r] = W[e] x[r] for the rows r of each expert e's segment -> bf16 [rows,N].

    x bf16 [rows,K]; weight bf16 [E,N,K], E <= 256, K and N multiples of 8.  efo i32 [E+1]: first row of each expert's segment, ascending;
    any rows, so that segments may follow one another without padding (0 and the cumulative counts), or start at multiples of 128 as the
    routing metadata leaves them, with counts i32 [E], the live rows at each segment's start (all without it).  Rows that are not live,
    those outside every segment among them, may hold anything: their outputs and gradients are zero, and they are no part of the
    weight's.  Without efo there is one weight ([1,N,K] or [N,K]), every row is live, and x may have leading dimensions.

    Sums are f32, results bf16.  Differentiable in x and weight; a weight's gradient is added to the parameter's f32 `main_grad` where it
    has one, else returned in bf16.  Gradients cannot be differentiated again, and there are no forward-mode
    derivatives."""
    ops.poll_status(x.device)                 # a device-side failure of an earlier call surfaces here, without a sync
    grad = torch.is_grad_enabled()
    if not x.is_cuda:
        _host.grouped_checked(x, weight, efo, counts)      # (which refuses it, by the arguments or for want of a GPU)
    if ops._recorder is None and not (grad and weight.requires_grad and getattr(_base_of(weight), "main_grad", None) is not None):
        return _host.grouped_call(x, weight, efo, counts, *ops.failure_words(x.device))
    rows, _ = _host.grouped_checked(x, weight, efo, counts)
    if grad and (x.requires_grad or weight.requires_grad):
        y = _GroupedLinear.apply(rows, weight, efo, counts)
    else:
        w = _weight16(weight)
        y = ops.grouped_rows(rows, w if w.ndim == 3 else w[None], efo, counts)
    return y if x.ndim == 2 else y.view(*x.shape[:-1], weight.shape[-2])
