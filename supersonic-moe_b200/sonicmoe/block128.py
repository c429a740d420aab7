"""FP8 products with one f32 scale per block of 128: activations in e4m3 with a scale for each row and 128 columns, weights with a
scale for each 128 x 128.  Beside the 1x32 MXFP8 path of the layer, for weights that come in this form; not part of the
reference signature.

A block's scale is a / 448 and its payload e4m3(x * (448 / a)) with a = max(max |x|, 2^-100).  Sizes are multiples of 8.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops
from .functional import _after_accumulate, _grad_target

_E4M3 = torch.float8_e4m3fn
FEW_ROWS = 64          # rows of one projection up to which its weights are the wide operand


def quantize_rows_block128(x: torch.Tensor, swiglu: bool = False):
    """bf16 [rows,K] -> (e4m3 [rows,K], scales f32 [rows,ceil(K/128)]).  `swiglu`: x is [rows,2K] with gate and up interleaved (what an
    up-projection leaves) and silu(gate) * up is what is quantised, without leaving the chip in between."""
    q, s = ops.quant128_rows(x.contiguous(), swiglu)
    return q.view(_E4M3), s


def quantize_weight_block128(w: torch.Tensor):
    """bf16 [E,N,K] (or [N,K]) -> (e4m3 of that shape, scales f32 [E,ceil(N/128),ceil(K/128)])."""
    q, s = _quantised(w)
    return (q.view(_E4M3), s) if w.ndim == 3 else (q[0].view(_E4M3), s[0])


def _quantised(w):
    return ops.quant128_weight(w.detach().contiguous().view(-1, *w.shape[-2:]))


def _fp8_weight(weight):
    """(payload [E,N,K], scales [E,..]) of a quantised weight given as a pair."""
    q, s = weight
    if q.ndim == 2:
        q, s = q[None], s[None]
    if q.ndim != 3 or q.element_size() != 1:
        raise ValueError(f"block128: a quantised weight is (e4m3 [E,N,K], scales), got {q.dtype} {tuple(q.shape)}")
    return q, s


def _forward(x, q, s, efo, counts):
    xq, xs = x
    if efo is None and xq.shape[0] <= FEW_ROWS:
        return ops.gemm128_few(xq, xs, q, s)
    return ops.gemm128_rows(xq, xs, q, s, efo, counts)


class _Block128Linear(torch.autograd.Function):
    """x [rows,K], weight bf16 [E,N,K] or [N,K], or None with (q, s) its quantised form."""

    @staticmethod
    def forward(ctx, x, weight, q, s, efo, counts):
        if weight is not None:
            q, s = _quantised(weight)
        xc = xcs = None
        if ctx.needs_input_grad[1]:            # the column form is what the weight gradient reads: half the bytes of x to keep
            xq, xs, xc, xcs = ops.quant128_dual(x, efo, counts)
        else:
            xq, xs = ops.quant128_rows(x)
        ctx.save_for_backward(q if ctx.needs_input_grad[0] else None, s if ctx.needs_input_grad[0] else None, xc, xcs, efo, counts)
        ctx.weight = weight
        return _forward((xq, xs), q, s, efo, counts)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        q, s, xc, xcs, efo, counts = ctx.saved_tensors
        dy = dy.contiguous()
        dx = dw = None
        if ctx.needs_input_grad[1]:
            dq, ds, dc, dcs = ops.quant128_dual(dy, efo, counts, with_rows=ctx.needs_input_grad[0])
        else:
            dq, ds = ops.quant128_rows(dy)
        if ctx.needs_input_grad[0]:
            dx = ops.gemm128_rows(dq, ds, q, s, efo, counts, b_mn=True)
        if ctx.needs_input_grad[1]:
            main_grad, base = _grad_target(ctx.weight, ctx.weight.shape)
            if main_grad is not None:
                ops.gemm128_wgrad(dc, dcs, xc, xcs, efo, counts, out=main_grad.view(-1, *main_grad.shape[-2:]), accumulate=True)
                _after_accumulate(base)
            else:
                dw = ops.gemm128_wgrad(dc, dcs, xc, xcs, efo, counts).view(ctx.weight.shape)
        return dx, dw, None, None, None, None


def block128_linear(x: torch.Tensor, weight, efo: torch.Tensor | None = None, counts: torch.Tensor | None = None) -> torch.Tensor:
    """y = x W^T by expert segments with both operands quantised in blocks of 128 -> bf16 [rows,N].

    x bf16 [rows,K]; weight either bf16 [E,N,K], quantised in the call and differentiable (its gradient goes to the parameter's f32
    `main_grad` where it has one, else it is returned in bf16), or the pair of `quantize_weight_block128`, made once and constant.
    efo i32 [E+1]: first row of each expert's segment, multiples of 128 as the routing metadata leaves them; counts i32 [E]: its
    live rows (all without it).  Rows that are not live, also those behind the last segment, are ignored: their outputs and
    gradients are zero.  Without efo there is one weight ([1,N,K] or [N,K]), every row is live, and x may have leading dimensions.

    The gradient of x is a product with the same payload; both gradients quantise dy, along its columns for x and along 128 rows
    for the weight."""
    if x.dtype != torch.bfloat16:
        raise ValueError(f"block128_linear: x is bf16, got {x.dtype}")
    ops.poll_status(x.device)                 # a device-side failure of an earlier call surfaces here, without a sync
    pair = isinstance(weight, (tuple, list))
    q = s = None
    if pair:
        q, s = _fp8_weight(weight)
        E, N, K = q.shape
    else:
        if weight.ndim not in (2, 3) or weight.dtype != torch.bfloat16:
            raise ValueError(f"block128_linear: the weight is bf16 [E,N,K], got {weight.dtype} {tuple(weight.shape)}")
        E, N, K = weight.shape if weight.ndim == 3 else (1, *weight.shape)
    if x.shape[-1] != K:
        raise ValueError(f"block128_linear: x has {x.shape[-1]} columns, the weight {K}")
    if efo is None and (E != 1 or counts is not None):
        raise ValueError("block128_linear: several experts, or counts, need efo")
    if efo is not None and x.ndim != 2:
        raise ValueError("block128_linear: x is [rows,K] where efo is given")
    rows = x.reshape(-1, K).contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (not pair and weight.requires_grad)):
        y = _Block128Linear.apply(rows, None if pair else weight, q, s, efo, counts)
    else:
        if not pair:
            q, s = _quantised(weight)
        y = _forward(ops.quant128_rows(rows.detach()), q, s, efo, counts)
    return y if x.ndim == 2 else y.view(*x.shape[:-1], N)


def _few_rows_per_expert(T, K, E):
    return T * K <= 16 * E or T <= FEW_ROWS


@torch.no_grad()
def block128_experts(x: torch.Tensor, topk_indices: torch.Tensor, topk_scores: torch.Tensor, w1_fp8, w2_fp8) -> torch.Tensor:
    """SwiGLU experts on routed tokens, inference: out[t] = sum_k scores[t,k] * W2[e] silu-gated(W1[e] x[t]), e = indices[t,k].

    x bf16 [T,H]; topk_indices [T,K] (-1: no expert in this slot; a token's experts distinct), topk_scores [T,K];
    w1_fp8, w2_fp8: pairs of `quantize_weight_block128` of W1 [E,2I,H] (gate and up rows interleaved) and W2 [E,H,I].  Returns bf16
    [T,H].  Both products leave bf16; what lies between is quantised in blocks of 128 like x.  No gradient flows."""
    if x.ndim != 2 or x.dtype != torch.bfloat16:
        raise ValueError(f"block128_experts: x is bf16 [T,H], got {x.dtype} {tuple(x.shape)}")
    ops.poll_status(x.device)
    (q1, s1), (q2, s2) = _fp8_weight(w1_fp8), _fp8_weight(w2_fp8)
    T, H = x.shape
    E, N1, I = q1.shape[0], q1.shape[1], q1.shape[1] // 2
    if q1.shape[2] != H or tuple(q2.shape) != (E, H, I) or N1 % 2:
        raise ValueError(f"block128_experts: x [{T},{H}] against W1 {tuple(q1.shape)} and W2 {tuple(q2.shape)}")
    if topk_indices.ndim != 2 or topk_indices.shape[0] != T or topk_scores.shape != topk_indices.shape:
        raise ValueError(f"block128_experts: indices {tuple(topk_indices.shape)} and scores {tuple(topk_scores.shape)} of {T} tokens")
    K = topk_indices.shape[1]
    if T == 0 or K == 0:
        return torch.zeros_like(x)
    idx = topk_indices.to(torch.int32).contiguous()
    md = ops.topk_metadata(idx, topk_scores.float().contiguous(), E, 128)
    rows, places, live = md["TKp_alloc"], md["s_reverse_scatter_idx"], md["naept"][-1:]
    few = _few_rows_per_expert(T, K, E)

    def product(a, b):
        if few:
            return ops.gemm128_few(*a, *b, md["efo"], md["counts"], live_rows=T * min(K, E))
        return ops.gemm128_rows(*a, *b, md["efo"], md["counts"], zero_rest=False)

    z = product(ops.quant128_rows_scatter(x.contiguous(), md["naept"], places, rows), (q1, s1))
    o = product(ops.quant128_rows(z, True, places, live), (q2, s2))
    return ops.combine(o, places, md["naept"], md["topk_scores"], T)
