"""The global norm of a model's gradients and their clipping, over `main_grad` accumulators and ordinary gradients alike, f32 and bf16
together.  Not part of the reference signature, which leaves both to its host framework.
"""
from __future__ import annotations

import math

import torch

from . import ops

_Parameter = torch.nn.Parameter


def _gradients(items, what):
    """Gradient tensors of parameters (f32 `main_grad` before `.grad`; those with neither left out), tensors as they are."""
    out = []
    for t in (items,) if isinstance(items, torch.Tensor) else items:
        if type(t) is not torch.Tensor and isinstance(t, _Parameter):
            g = getattr(t, "main_grad", None)
            t = t.grad if g is None else g
            if t is None:
                continue
        out.append(t)
    if not out:
        raise ValueError(f"{what}: no gradients")
    return out


def gradient_norm(gradients) -> torch.Tensor:
    """sqrt(sum of the squares of all values of all gradients) -> f32 [] on their GPU.

    gradients: tensors, f32 or bf16, of any shapes, or parameters, which stand for their `main_grad`, else their `.grad` (those with
    neither are left out).  f32 sums of a few values, f64 beyond, in one order.  Nothing is copied to the host.  Across ranks that hold
    different parameters the squares of their norms add up: all-reduce those and hand the root to `clip_gradients(norm=...)`."""
    grads = _gradients(gradients, "gradient_norm")
    return ops.gradient_norm([g if g.is_contiguous() else g.contiguous() for g in grads])


def clip_gradients(gradients, max_norm: float, *, norm: torch.Tensor | None = None, out=None) -> torch.Tensor:
    """gradients *= min(1, max_norm / (n + 1e-6)), n their norm, which is returned (f32 [], before clipping, on their GPU).

    gradients: as `gradient_norm` takes them, each once.  `norm`: f32 [], instead of theirs (that of all ranks).  `out`: contiguous
    f32 or bf16 tensors of the gradients' shapes, one for each, which receive the results (accumulators in f32, gradients for the
    optimizer in bf16, from one pass); the gradients stay as they are then.  Without it they change in place, and where nothing is to
    be clipped nothing is written.  A norm of NaN makes every result NaN, an infinite one 0 (NaN where the gradient is infinite)."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_gradients: max_norm={max_norm}")
    grads = _gradients(gradients, "clip_gradients")
    if norm is not None and (norm.numel() != 1 or norm.dtype != torch.float32 or norm.device != grads[0].device):
        raise ValueError(f"clip_gradients: the norm is one f32 on {grads[0].device}, got {norm.dtype} {tuple(norm.shape)} on {norm.device}")
    dense = [g if g.is_contiguous() else g.contiguous() for g in grads]
    if out is None:
        _once(dense, "gradients")
        n = ops.gradient_clip(dense, max_norm, norm)
        for g, d in zip(grads, dense):
            if g is not d:
                g.detach().copy_(d)
        _written(grads)
        return n
    out = list(out)
    if len(out) != len(grads):
        raise ValueError(f"clip_gradients: {len(out)} outputs for {len(grads)} gradients")
    for g, o in zip(grads, out):
        if o.shape != g.shape or not o.is_contiguous():
            raise ValueError(f"clip_gradients: outputs are contiguous and of their gradients' shapes, got {tuple(o.shape)} for {tuple(g.shape)}")
    _once(out, "outputs")
    ins = {g.data_ptr(): g for g in dense if g.numel()}
    for g, o in zip(dense, out):
        if o.numel() and (ins.get(o.data_ptr(), g) is not g or (o.data_ptr() == g.data_ptr() and o.dtype != g.dtype)):
            raise ValueError("clip_gradients: an output lies where another gradient does")
    n = ops.gradient_clip(dense, max_norm, norm, out)
    _written(out)
    return n


def _once(tensors, what):
    at = [t.data_ptr() for t in tensors if t.numel()]
    if len(set(at)) != len(at):
        raise ValueError(f"clip_gradients: one of the {what} is given twice")


def _written(tensors):
    """Autograd sees that they are other tensors now (those of inference mode have nothing to see it by)."""
    torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])
