"""Group-limited routing against its definition in 64 bits: choices are equal, scores and gradients within roundings."""
import math

import pytest
import torch

from oracle import group_routing as G

pytestmark = pytest.mark.gpu
DEV = "cuda"
# exp, its argument's rounding (at most 30 here), the sum of E <= 1024 terms over 32 lanes, quotients: counted in roundings of f32
SCORE_TOL = 128 * 2.0 ** -24


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    return m


def call(sonicmoe, logits, K, bias=None, **rule):
    return sonicmoe.group_limited_routing(logits, K, bias=bias, score="softmax" if rule.pop("softmax", False) else "sigmoid", **rule)


def check(sonicmoe, logits, K, bias=None, groups=1, top_groups=1, group_score=2, softmax=False, normalize=True, scale=1.0, seed=0):
    """Choices, scores and gradient of one batch."""
    x = logits.to(DEV).requires_grad_(True)
    rule = dict(groups=groups, top_groups=top_groups, group_score=group_score, normalize=normalize, scale=scale)
    scores, idx = call(sonicmoe, x, K, None if bias is None else bias.to(DEV), softmax=softmax, **rule)
    ref, ref_idx = G.route(logits, K, bias, softmax=softmax, **rule)
    assert scores.dtype == torch.float32 and idx.dtype == torch.int32
    assert torch.equal(idx.cpu(), ref_idx)
    assert ((scores.detach().cpu().double() - ref).abs() <= SCORE_TOL * ref.abs() + 1e-37).all()
    g = torch.randn(logits.shape[0], K, generator=torch.Generator().manual_seed(seed))
    grad, = torch.autograd.grad(scores, x, g.to(DEV))
    want = G.route_grad(logits, ref_idx, g, softmax, normalize, scale)
    # what the terms of an element's gradient add up to in magnitude
    s = G.all_scores(logits.double(), softmax)
    real = ref_idx >= 0
    at = ref_idx.clamp(min=0).long()
    sk = torch.where(real, s.gather(1, at), 0.0)
    gk = torch.where(real, g.double().abs() * abs(scale), 0.0)
    D = sk.sum(-1, keepdim=True) + 1e-20 if normalize else torch.ones(len(s), 1, dtype=torch.float64)
    dk = gk / D + ((gk * sk).sum(-1, keepdim=True) / D ** 2 if normalize else 0)
    mag = torch.zeros_like(s).scatter_add_(1, at, torch.where(real, dk, 0.0)) + ((dk * sk).sum(-1, keepdim=True) if softmax else 0)
    tol = SCORE_TOL * s * mag + (2.0 ** -8 * want.abs() if logits.dtype == torch.bfloat16 else 0) + 1e-30
    assert grad.dtype == logits.dtype
    assert ((grad.cpu().double() - want).abs() <= tol).all()
    return scores, idx


def randn(T, E, seed, dtype=torch.float32, scale=1.5):
    return (torch.randn(T, E, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


@pytest.mark.parametrize("E,K,groups,top_groups", [(1, 1, 1, 1), (8, 2, 1, 1), (8, 8, 4, 4), (37, 5, 1, 1), (60, 6, 5, 3), (64, 8, 8, 4),
                                                   (96, 7, 32, 9), (128, 8, 8, 4), (160, 6, 8, 3), (256, 8, 8, 4), (256, 32, 4, 1),
                                                   (320, 8, 5, 2), (1000, 8, 8, 3), (1024, 32, 32, 16)])
@pytest.mark.parametrize("softmax", [False, True])
def test_choices_scores_and_gradients(sonicmoe, E, K, groups, top_groups, softmax):
    for i, (T, dtype, with_bias, group_score, normalize) in enumerate(
            [(1, torch.float32, True, 2, True), (67, torch.bfloat16, True, 2, False), (66, torch.bfloat16, False, 1, True),
             (65, torch.float32, False, 2, True)]):
        bias = randn(1, E, 100 + i)[0] * (0.05 if softmax else 0.3) if with_bias else None
        check(sonicmoe, randn(T, E, 10 * i + E, dtype), K, bias, groups, top_groups, group_score, softmax, normalize, 2.5)


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
def test_equal_and_nearly_equal_scores(sonicmoe, softmax, with_bias):
    """Rows of one value, of few values, of values one rounding apart; a bias of zeros, of few values, and one that undoes the scores."""
    E, K = 256, 8
    g = torch.Generator().manual_seed(3)
    one = torch.full((4, E), 0.3)
    few = torch.randint(-2, 3, (24, E), generator=g).float()
    near = (1.0 + torch.randint(0, 4, (24, E), generator=g).float() * 2.0 ** -23)
    logits = torch.cat([one, few, near, torch.zeros(2, E)])
    biases = [None]
    if with_bias:
        biases = [torch.zeros(E), torch.randint(0, 3, (E,), generator=g) * 0.25,
                  0.5 - G.all_scores(few[:1].double(), softmax)[0].float()]
    for b in biases:
        for group_score in (1, 2):
            check(sonicmoe, logits, K, b, 8, 4, group_score, softmax)
            check(sonicmoe, logits.bfloat16(), K, b, 1, 1, group_score, softmax)


@pytest.mark.parametrize("softmax", [False, True])
def test_closed_experts_and_padded_tokens(sonicmoe, softmax):
    E, K = 64, 6
    logits = randn(40, E, 5)
    closed = torch.rand(40, E, generator=torch.Generator().manual_seed(6)) < torch.linspace(0, 1, 40)[:, None]
    logits[closed] = -math.inf
    logits[-3:] = -math.inf
    logits[7] = -math.inf
    logits[7, 33] = 0.25                                      # one open expert
    bias = randn(1, E, 8)[0] * 0.2
    for groups, top in ((1, 1), (8, 3)):
        for b in (None, bias):
            scores, idx = check(sonicmoe, logits, K, b, groups, top, 2, softmax)
            assert (idx[-3:] == -1).all() and (scores[-3:] == 0).all()
            assert idx[7].tolist() == [33] + [-1] * 5


def test_nan_ranks_lowest_and_large_values_are_kept_apart(sonicmoe):
    E, K = 32, 4
    logits = randn(6, E, 9)
    logits[0, ::2] = math.nan
    logits[1] = math.nan
    logits[2, 5] = math.inf
    logits[3] *= 20                                           # sigmoid is 1 but for a few units of 2^-53
    bias = torch.zeros(E)
    bias[3], bias[4], bias[9] = -math.inf, math.nan, 1e30
    for b in (None, bias):
        _, idx = call(sonicmoe, logits.to(DEV), K, None if b is None else b.to(DEV), groups=4, top_groups=2)
        _, ref = G.route(logits, K, b, 4, 2)
        assert torch.equal(idx.cpu(), ref)
        assert all(len(set(r)) == K and min(r) >= 0 and max(r) < E for r in idx.tolist())


def test_gradient_against_differences(sonicmoe):
    T, E, K = 5, 40, 4
    logits, g = randn(T, E, 11), torch.randn(T, K, generator=torch.Generator().manual_seed(12))
    for softmax, normalize in ((False, True), (True, True), (True, False)):
        x = logits.to(DEV).requires_grad_(True)
        scores, idx = call(sonicmoe, x, K, softmax=softmax, normalize=normalize, scale=1.5)
        grad, = torch.autograd.grad(scores, x, g.to(DEV))
        h = 1e-5
        for e in range(E):
            d = torch.zeros(T, E, dtype=torch.float64)
            d[:, e] = h
            f = [(G.scores_of(logits.double() + w * d, idx.cpu(), softmax, normalize, 1.5) * g.double()).sum(-1) for w in (1, -1)]
            # the difference quotient is off by h^2 times the third derivative, at most a few units here
            assert ((f[0] - f[1]) / (2 * h) - grad[:, e].cpu().double()).abs().max() <= 1e-5


def test_non_contiguous_logits_and_gradients(sonicmoe):
    base = randn(16, 128, 13).to(DEV)
    x = base[:, ::2].detach().requires_grad_(True)
    scores, idx = call(sonicmoe, x, 4)
    assert torch.equal(idx, call(sonicmoe, base[:, ::2].contiguous(), 4)[1])
    g = torch.randn(4, 16, device=DEV).T
    a, = torch.autograd.grad(scores, x, g, retain_graph=True)
    b, = torch.autograd.grad(scores, x, g.contiguous())
    assert torch.equal(a, b)
    c, = torch.autograd.grad(call(sonicmoe, x, 4)[0].sum(), x)          # a gradient that is one value, broadcast
    assert c.shape == x.shape


def test_no_tokens_and_replays(sonicmoe):
    scores, idx = call(sonicmoe, torch.empty(0, 16, device=DEV), 4)
    assert scores.shape == idx.shape == (0, 4)
    x, bias = randn(33, 64, 14).to(DEV), torch.zeros(64, device=DEV)
    call(sonicmoe, x, 4, bias, groups=8, top_groups=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scores, idx = call(sonicmoe, x, 4, bias, groups=8, top_groups=2)
    x.copy_(randn(33, 64, 15))
    graph.replay()
    want = call(sonicmoe, x, 4, bias, groups=8, top_groups=2)
    assert torch.equal(idx, want[1]) and torch.equal(scores, want[0])


@pytest.mark.parametrize("softmax", [False, True])
@pytest.mark.parametrize("K", [1, 4])
def test_gradient_of_normalised_weights_that_cannot_move(sonicmoe, softmax, K):
    """One weight, or all with the same gradient: their sum does not move (1e-20 is no part of these sums in f32)."""
    x = randn(33, 24, 7).to(DEV).requires_grad_(True)
    scores, _ = call(sonicmoe, x, K, softmax=softmax, scale=2.0)
    grad, = torch.autograd.grad(scores, x, torch.full_like(scores, 1.5))
    assert (grad == 0).all()


def test_gradient_where_the_sum_is_as_small_as_what_is_added_to_it(sonicmoe):
    """s / (s + 1e-20) with s about 1e-20: 1e-20 g s (1 - s) / (s + 1e-20)^2 at the expert chosen."""
    x = (randn(40, 24, 8) - 46.0).to(DEV).requires_grad_(True)
    scores, idx = call(sonicmoe, x, 1)
    grad, = torch.autograd.grad(scores, x, torch.full_like(scores, 1.5))
    s = torch.sigmoid(x.detach().cpu().double())
    want = torch.zeros_like(s).scatter_(1, idx.cpu().long(), 1.5)
    want = want * 1e-20 * s * (1 - s) / (s + 1e-20) ** 2
    assert want.abs().max() > 0.1
    # exp of 46 +- 6: its argument's rounding is 2^-24 of at most 52, and the score enters three times
    assert ((grad.cpu().double() - want).abs() <= (3 * 52 + 64) * 2.0 ** -24 * want).all()
