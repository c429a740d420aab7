"""The global norm of a model's gradients and their clipping, over `main_grad` accumulators and ordinary gradients alike, f32 and bf16
together.  Not part of the reference signature, which leaves both to its host framework.
"""
from __future__ import annotations

import torch

from . import ops


def gradient_norm(gradients) -> torch.Tensor:
    """sqrt(sum of the squares of all values of all gradients) -> f32 [] on their GPU.

    gradients: tensors, f32 or bf16, of any shapes, or parameters, which stand for their `main_grad`, else their `.grad` (those with
    neither are left out).  f32 sums of a few values, f64 beyond, in one order.  Nothing is copied to the host, and no gradient flows through it.  Across ranks that hold
    different parameters the squares of their norms add up: all-reduce those and hand the root to `clip_gradients(norm=...)`."""
    return ops.gradient_norm(gradients)


def clip_gradients(gradients, max_norm: float, *, norm: torch.Tensor | None = None, out=None) -> torch.Tensor:
    """gradients *= min(1, max_norm / (n + 1e-6)), n their norm, which is returned (f32 [], before clipping, on their GPU).

    gradients: as `gradient_norm` takes them, none overlapping another.  `norm`: f32 [], instead of theirs (that of all ranks).  `out`:
    contiguous f32 or bf16 tensors of the gradients' shapes, one for each (a single one as the gradients), which receive the results (accumulators in f32, gradients
    for the optimizer in bf16, from one pass); the gradients stay as they are then.  An output may be its own gradient and lies apart
    from every other one.  Without `out` they change in place (an expanded gradient is refused, a strided one goes through a copy and is
    written always), and where nothing is to be clipped nothing else is written.  A norm of NaN makes every result NaN, an infinite one 0
    (NaN where the gradient is infinite)."""
    return ops.clip_gradients(gradients, float(max_norm), norm, out)
