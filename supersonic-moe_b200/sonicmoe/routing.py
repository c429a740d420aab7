"""Routers beside the layer's own softmax top-k: `group_limited_routing` makes the [T,K] tables that `run_sonic_moe` and
`block128_experts` take (up to 16 experts a token, of 256 there), `token_rounding_routing` (score, token, expert) pair lists for
`moe_general_routing_inputs`.

`token_rounding_routing` restates the token-rounding router of the reference's benchmark
(benchmarks/moe-token-rounding.py:139-181): a token-choice top-K pass fixes each expert's load, the load is rounded
to a multiple of the GEMM row tile, and an expert-choice pass over the combined scores (top-K picks first, then the
rest by score) fills or trims every expert to exactly that many tokens.  With every count a multiple of the tile no
expert segment needs pad rows.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import ops
from .count_cumsum import count_cumsum


class _GroupLimitedRouting(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, K, rule):
        scores, idx = ops.group_routing(logits, K, *rule)
        ctx.save_for_backward(logits, idx)
        ctx.rule = rule[4:]                                  # softmax, normalize, scale
        ctx.mark_non_differentiable(idx)
        return scores, idx

    @staticmethod
    @once_differentiable
    def backward(ctx, dscores, _didx):
        logits, idx = ctx.saved_tensors
        if dscores.dtype != torch.float32 or not dscores.is_contiguous():
            dscores = dscores.float().contiguous()
        return ops.group_routing_bwd(logits, idx, dscores, *ctx.rule), None, None


def group_limited_routing(router_logits: torch.Tensor, K: int, *, score: str = "sigmoid", bias: torch.Tensor | None = None,
                          groups: int = 1, top_groups: int | None = None, group_score: int = 2, normalize: bool = True,
                          scale: float = 1.0):
    """Router logits [T,E] (f32 or bf16) -> (scores f32 [T,K], expert indices i32 [T,K]), differentiable in the logits.

    An expert's score is the sigmoid of its logit, or (`score="softmax"`) its softmax over all experts.  Experts are chosen by score +
    `bias` (f32 [E], a constant that balances their load; it has no part in the scores returned).  With `groups` > 1 the experts
    are that many runs of neighbours, a group ranks by the sum of its `group_score` (1 or 2) best experts, and only those of the
    `top_groups` best groups are eligible.  The K best, in descending order, the first of equals first, get scale * score / sum of
    the K scores (`normalize`) or scale * score.

    A logit of -inf closes its expert; a row with fewer than K open experts ends in slots of index -1 and score 0 (the layer's
    mark of a slot without an expert), so that a padded token is a row of -inf.  NaN ranks lowest.  The selection is that of 64-bit
    arithmetic: it does not depend on how an exponential is rounded.  A bias of -inf makes its expert the last choice, and one of
    two best experts that has it its group, without closing them.  E <= 1024, K <= 32, groups <= 32 (the layer and
    `block128_experts` take tables of K <= 16, the latter of E <= 256)."""
    if score not in ("sigmoid", "softmax"):
        raise ValueError(f"score={score!r}: 'sigmoid' or 'softmax'")
    if router_logits.ndim != 2 or router_logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"router logits are f32 or bf16 [T,E], got {router_logits.dtype} {tuple(router_logits.shape)}")
    E = router_logits.shape[1]
    top_groups = groups if top_groups is None else top_groups
    if not (1 <= groups <= 32 and E % groups == 0 and 1 <= top_groups <= groups):
        raise ValueError(f"groups={groups}, top_groups={top_groups}: at most 32 groups that divide {E} experts evenly")
    if not (1 <= E <= 1024 and 1 <= K <= min(32, top_groups * (E // groups))):
        raise ValueError(f"K={K}: 1 to 32, at most the {top_groups * (E // groups)} experts of the groups chosen (E={E}, at most 1024)")
    if group_score not in (1, 2):
        raise ValueError(f"group_score={group_score}: 1 or 2")
    if bias is not None:
        if bias.shape != (E,):
            raise ValueError(f"bias {tuple(bias.shape)}: one value for each of {E} experts")
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.detach().float().contiguous()
    rule = (bias, groups, top_groups, group_score, score == "softmax", bool(normalize), float(scale))
    logits = router_logits if router_logits.is_contiguous() else router_logits.contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        return _GroupLimitedRouting.apply(logits, K, rule)
    return ops.group_routing(logits, K, *rule)


def token_rounding_routing(router_logits: torch.Tensor, K: int, Mtile: int = 128, routing: str = "nr"):
    """router_logits [T,E] -> (scores of the selected pairs [nnz], token_indices [nnz] ascending, expert_indices
    [nnz]).  routing: "down" / "up" / "nr" (nearest) rounding of each expert's top-K load to a multiple of Mtile."""
    T, E = router_logits.shape
    dev = router_logits.device
    scores = F.softmax(router_logits, dim=-1, dtype=torch.float32)
    topk_values, topk_indices = scores.topk(K, dim=-1)
    flat = topk_indices.reshape(-1).to(torch.int32).contiguous()
    if flat.is_cuda and E % 4 == 0:
        freq = count_cumsum(flat, E, do_cumsum=False)
    else:
        freq = torch.bincount(flat.long(), minlength=E).to(torch.int32)
    if routing == "down":
        rounded = torch.div(freq, Mtile, rounding_mode="floor") * Mtile
    elif routing == "up":
        rounded = torch.div(freq + Mtile - 1, Mtile, rounding_mode="floor") * Mtile
    elif routing == "nr":
        rounded = torch.round(freq.float() / Mtile).to(torch.int32) * Mtile
    else:
        raise NotImplementedError(f"routing={routing!r}")
    rounded = rounded.clamp(max=T)
    topk_values = topk_values / topk_values.sum(dim=-1, keepdim=True)
    scores = scores.scatter(-1, topk_indices, topk_values)
    # expert-choice order: a token's top-K picks rank above everything else, each class by score
    combined = scores.detach() - 1
    combined.scatter_(1, topk_indices, topk_values.detach())
    order = combined.argsort(dim=0, descending=True).int()                       # [T,E]: per expert, tokens by rank
    keep = torch.arange(T, device=dev, dtype=torch.int32)[:, None] < rounded[None, :]
    token_indices = order[keep]
    expert_indices = torch.arange(E, device=dev, dtype=torch.int32)[None, :].expand(T, -1)[keep]
    by_token = token_indices.argsort(stable=True)
    token_indices, expert_indices = token_indices[by_token], expert_indices[by_token]
    return scores[token_indices.long(), expert_indices.long()].contiguous(), token_indices, expert_indices
