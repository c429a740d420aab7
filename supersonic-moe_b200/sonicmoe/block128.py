"""FP8 products with one f32 scale per block of 128: activations in e4m3 with a scale for each row and 128 columns, weights with a
scale for each 128 x 128.  Beside the 1x32 MXFP8 path of the layer, for weights that come in this form; not part of the
reference signature.

A block's scale is a / 448 and its payload e4m3(x * (448 / a)) with a = max(max |x|, 2^-100).  Sizes are multiples of 8; where the
columns are no multiple of 16 a payload is a view whose rows start on 16-byte boundaries.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops
from .functional import _after_accumulate, _grad_target

_E4M3 = torch.float8_e4m3fn


def _dense(t: torch.Tensor) -> torch.Tensor:
    """Contiguous, from a 16-byte boundary on (a view into a larger buffer need not be)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def quantize_rows_block128(x: torch.Tensor, swiglu: bool = False):
    """bf16 [rows,K] -> (e4m3 [rows,K], scales f32 [rows,ceil(K/128)]).  `swiglu`: x is [rows,2K] with gate and up interleaved (what an
    up-projection leaves) and silu(gate) * up is what is quantised, without leaving the chip in between; the payload is that of
    64-bit arithmetic (but for e4m3's subnormals, and gates below -16)."""
    q, s = ops.quant128_rows(_dense(x), swiglu)
    return q.view(_E4M3), s


def quantize_weight_block128(w: torch.Tensor):
    """bf16 [E,N,K] (or [N,K]) -> (e4m3 of that shape, scales f32 [E,ceil(N/128),ceil(K/128)])."""
    if w.ndim not in (2, 3):
        raise ValueError(f"quantize_weight_block128: the weight is bf16 [E,N,K] or [N,K], got {w.dtype} {tuple(w.shape)}")
    q, s = ops.quant128_weight(_dense(w.detach()).view(-1, *w.shape[-2:]))
    return (q.view(_E4M3), s) if w.ndim == 3 else (q[0].view(_E4M3), s[0])


def _fp8_weight(weight, what):
    """(payload [E,N,K], scales [E,N/128,K/128]) of a quantised weight given as a pair."""
    q, s = weight
    if q.ndim == 2:
        q, s = q[None], s[None]
    if q.ndim != 3:
        raise ValueError(f"{what}: a quantised weight is (e4m3 [E,N,K], scales), got {q.dtype} {tuple(q.shape)}")
    ops.check_payload(q, what)
    E, N, K = q.shape
    if s.dtype != torch.float32 or s.shape != (E, (N + 127) // 128, (K + 127) // 128) or not s.is_contiguous():
        raise ValueError(f"{what}: the scales of {tuple(q.shape)} are f32 [{E},{(N + 127) // 128},{(K + 127) // 128}], got {s.dtype} "
                         f"{tuple(s.shape)}")
    return q, s


class _Block128Linear(torch.autograd.Function):
    """x [rows,K]; weight bf16 [E,N,K] or [N,K], or None; `of` = (its quantised form or None twice, efo, counts, E, N, K)."""

    @staticmethod
    def forward(ctx, x, weight, of):
        q, s, efo, counts, E, N, K = of
        dx, dw, _ = ctx.needs_input_grad
        flags = (ops.B128_QUANT_W if weight is not None else 0) | (ops.B128_DW if dw else 0)
        y, saved = ops.block128_linear(x, q if weight is None else _dense(weight), s, efo, counts, E, N, K, flags)
        ctx.save_for_backward(q, s, efo, counts, saved)
        ctx.of = (E, N, K, flags | (ops.B128_DX if dx else 0))
        ctx.weight = weight if dw else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        q, s, efo, counts, saved = ctx.saved_tensors
        w, main_grad = ctx.weight, None
        if w is not None:
            main_grad, base = _grad_target(w, w.shape)
        dx, dw = ops.block128_linear_bwd(_dense(dy), q, s, efo, counts, saved, *ctx.of, main_grad)
        if main_grad is not None:
            _after_accumulate(base)
        return dx, None if dw is None else dw.view(w.shape), None


def block128_linear(x: torch.Tensor, weight, efo: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> torch.Tensor:
    """y = x W^T by expert segments with both operands quantised in blocks of 128 -> bf16 [rows,N].

    x bf16 [rows,K]; weight either bf16 [E,N,K], quantised in the call and differentiable (its gradient goes to the parameter's f32
    `main_grad` where it has one, else it is returned in bf16), or the pair of `quantize_weight_block128`, made once and constant.
    efo i32 [E+1]: first row of each expert's segment, multiples of 128 as the routing metadata leaves them; counts i32 [E]: its
    live rows (all without it).  Rows that are not live, also those behind the last segment, are ignored: their outputs and
    gradients are zero.  Without efo there is one weight ([1,N,K] or [N,K]), every row is live, and x may have leading dimensions.

    The gradient of x is a product with the same payload; both gradients quantise dy, along its columns for x and along 128 rows
    for the weight.  Gradients cannot be differentiated again."""
    if x.dtype != torch.bfloat16:
        raise ValueError(f"block128_linear: x is bf16, got {x.dtype}")
    ops.poll_status(x.device)                 # a device-side failure of an earlier call surfaces here, without a sync
    pair = isinstance(weight, (tuple, list))
    q = s = None
    if pair:
        q, s = _fp8_weight(weight, "block128_linear")
        E, N, K = q.shape
        weight = None
    else:
        if weight.ndim not in (2, 3) or weight.dtype != torch.bfloat16:
            raise ValueError(f"block128_linear: the weight is bf16 [E,N,K], got {weight.dtype} {tuple(weight.shape)}")
        E, N, K = weight.shape if weight.ndim == 3 else (1, *weight.shape)
    if x.shape[-1] != K:
        raise ValueError(f"block128_linear: x has {x.shape[-1]} columns, the weight {K}")
    if efo is not None and x.ndim != 2:
        raise ValueError("block128_linear: x is [rows,K] where efo is given")
    ops.check_segments(efo, counts, E, "block128_linear")
    rows = _dense(x if x.ndim == 2 else x.reshape(-1, K))
    if torch.is_grad_enabled() and (x.requires_grad or (not pair and weight.requires_grad)):
        y = _Block128Linear.apply(rows, weight, (q, s, efo, counts, E, N, K))
    elif pair:
        y = ops.block128_linear(rows, q, s, efo, counts, E, N, K, 0)[0]
    else:
        y = ops.block128_linear(rows, _dense(weight), None, efo, counts, E, N, K, ops.B128_QUANT_W)[0]
    return y if x.ndim == 2 else y.view(*x.shape[:-1], N)


def block128_experts(x: torch.Tensor, topk_indices: torch.Tensor, topk_scores: torch.Tensor, w1_fp8, w2_fp8) -> torch.Tensor:
    """SwiGLU experts on routed tokens, inference: out[t] = sum_k scores[t,k] W2[e] (silu(gate) * up), gate and up the interleaved rows
    of W1[e] x[t], e = indices[t,k].

    x bf16 [T,H]; topk_indices [T,K] (-1: no expert in this slot; one that a token names twice counts twice), topk_scores [T,K];
    w1_fp8, w2_fp8: pairs of `quantize_weight_block128` of W1 [E,2I,H] and W2 [E,H,I], E <= 256, K <= 16 (a checkpoint that holds gate and
    up as two matrices has other blocks than W1: it is put together in bf16 and quantised).  Returns bf16 [T,H].  Both products
    leave bf16; what lies between is quantised in blocks of 128 like x, as `quantize_rows_block128` does it.  No gradient flows."""
    if x.ndim != 2 or x.dtype != torch.bfloat16:
        raise ValueError(f"block128_experts: x is bf16 [T,H], got {x.dtype} {tuple(x.shape)}")
    ops.poll_status(x.device)
    (q1, s1), (q2, s2) = _fp8_weight(w1_fp8, "block128_experts"), _fp8_weight(w2_fp8, "block128_experts")
    T, H = x.shape
    E, I = q1.shape[0], q1.shape[1] // 2
    if q1.shape[2] != H or q2.shape != (E, H, I) or q1.shape[1] % 2:
        raise ValueError(f"block128_experts: x [{T},{H}] against W1 {tuple(q1.shape)} and W2 {tuple(q2.shape)}")
    if topk_indices.ndim != 2 or topk_indices.shape[0] != T or topk_scores.shape != topk_indices.shape:
        raise ValueError(f"block128_experts: indices {tuple(topk_indices.shape)} and scores {tuple(topk_scores.shape)} of {T} tokens")
    if T == 0 or topk_indices.shape[1] == 0:
        return torch.zeros_like(x)
    return ops.block128_experts(_dense(x.detach()), topk_indices.to(torch.int32).contiguous(),
                                topk_scores.detach().float().contiguous(), q1, s1, q2, s2, E, I)
