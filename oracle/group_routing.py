"""Group-limited routing on CPU in 64 bits, one row at a time as the definition reads."""
import math

import torch


def choose(logits, bias, K, groups, top_groups, group_score, softmax):
    """Chosen experts of one row, -1 beyond the open ones."""
    x = logits.double()
    E = x.numel()
    n = E // groups
    s = all_scores(x[None], softmax)[0]
    c = (s + bias.double()) if bias is not None else s
    clean = lambda v: -1.7976931348623157e308 if math.isnan(v) else min(max(v, -1.7976931348623157e308), 1.7976931348623157e308)
    c = [clean(float(v)) for v in c]
    order = c if bias is not None else [clean(float(v)) for v in x]
    by = order if bias is None and group_score == 1 else c
    is_open = [float(v) != -math.inf for v in x]
    if top_groups < groups:
        rank = []
        for g in range(groups):
            best = sorted((by[e] for e in range(g * n, g * n + n) if is_open[e]), reverse=True)[:group_score]
            rank.append((0 if best else 1, -sum(best), g))
        keep = {g for _, _, g in sorted(rank)[:top_groups]}
    else:
        keep = set(range(groups))
    able = sorted((-order[e], e) for e in range(E) if is_open[e] and e // n in keep)
    out = [e for _, e in able[:K]]
    return out + [-1] * (K - len(out))


def all_scores(x, softmax):
    """Scores of logits [T,E]; a closed expert has 0 and passes no gradient on."""
    if not softmax:
        return torch.sigmoid(x)
    closed = torch.isinf(x) & (x < 0)
    zero = torch.zeros((), dtype=x.dtype)
    top = x.detach().amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top) & (top < 0), zero, top)
    e = torch.where(closed, zero, torch.exp(torch.where(closed, top, x) - top))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-300)


def scores_of(x, idx, softmax, normalize, scale):
    """Scores in 64 bits of given choices [T,K], differentiable in x."""
    real = idx >= 0
    s = all_scores(x, softmax).gather(1, idx.clamp(min=0).long())
    s = torch.where(real, s, torch.zeros((), dtype=x.dtype))
    return scale * s / (s.sum(-1, keepdim=True) + 1e-20) if normalize else scale * s


def route(logits, K, bias=None, groups=1, top_groups=1, group_score=2, softmax=False, normalize=True, scale=1.0):
    idx = torch.tensor([choose(r, bias, K, groups, top_groups, group_score, softmax) for r in logits],
                       dtype=torch.int32).reshape(len(logits), K)
    return scores_of(logits.double(), idx, softmax, normalize, scale), idx


def route_grad(logits, idx, dscores, softmax, normalize, scale):
    x = logits.double().requires_grad_(True)
    return torch.autograd.grad(scores_of(x, idx, softmax, normalize, scale), x, dscores.double())[0]
