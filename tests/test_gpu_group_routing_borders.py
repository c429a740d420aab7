"""Group-limited routing where a group's score is made of values far larger than itself, or of a bias that is infinite: the choice is
that of 64 bits there too."""
import math

import pytest
import torch

from oracle import group_routing as G

pytestmark = pytest.mark.gpu
DEV = "cuda"
LOWEST = torch.finfo(torch.float32).min


@pytest.fixture(scope="module")
def sonicmoe():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import sonicmoe as m
    return m


def same_choice(sonicmoe, logits, K, bias, groups, top_groups, group_score, softmax):
    b = None if bias is None else bias.to(DEV)
    _, idx = sonicmoe.group_limited_routing(logits.to(DEV), K, score="softmax" if softmax else "sigmoid", bias=b, groups=groups,
                                            top_groups=top_groups, group_score=group_score)
    _, ref = G.route(logits, K, bias, groups, top_groups, group_score, softmax)
    assert torch.equal(idx.cpu(), ref)


# (E, groups): two lanes a group, four, several experts a lane, and sizes that no power of two divides
TABLES = [(8, 4), (64, 8), (256, 8), (12, 4), (60, 5), (1000, 8)]


def test_an_expert_switched_off_by_its_bias(sonicmoe):
    """Its group scores as low as it does: the other groups come first."""
    logits = torch.tensor([[3, 0, -2, -2.1, -2.2, -2.3, -2.4, -2.5]])
    bias = torch.zeros(8)
    bias[1] = -math.inf
    for softmax in (False, True):
        same_choice(sonicmoe, logits, 2, bias, 4, 2, 2, softmax)
    assert G.route(logits, 2, bias, 4, 2, 2, False)[1].tolist() == [[2, 3]]


@pytest.mark.parametrize("E,groups", TABLES)
@pytest.mark.parametrize("group_score", [1, 2])
@pytest.mark.parametrize("softmax", [False, True])
def test_groups_of_one_expert_or_none_that_its_bias_leaves(sonicmoe, E, groups, group_score, softmax):
    n, g = E // groups, torch.Generator().manual_seed(E)
    logits = torch.randn(40, E, generator=g)
    logits[30:][torch.rand(10, E, generator=g) < 0.5] = -math.inf
    logits[38, :n] = -math.inf                                # a closed group beside those that the bias leaves nothing of
    for off in (-math.inf, LOWEST):
        bias = torch.randn(E, generator=g) * 0.1
        bias[1:n] = off                                       # one is left of the first group, none of the second
        bias[n:2 * n] = off
        bias[2 * n + 1::2] = off                              # and half of the others
        for top in (1, groups // 2, groups - 1):
            same_choice(sonicmoe, logits, min(3, top * n), bias, groups, top, group_score, softmax)


@pytest.mark.parametrize("E,groups", TABLES)
@pytest.mark.parametrize("a", [10.0, 100.0, 1e4])
@pytest.mark.parametrize("softmax", [False, True])
def test_two_large_biases_that_cancel_in_a_group(sonicmoe, E, groups, a, softmax):
    """The scores' sum is near 1 but was rounded at the size of the biases.  Logits in steps of what that rounding is."""
    n, g = E // groups, torch.Generator().manual_seed(int(a) + E)
    bias = torch.full((groups, n), -a)
    bias[:, 0] = a
    wide = E if softmax else 1                                # a softmax score is 1 / E here
    logits = torch.randint(0, 16, (200, E), generator=g) * (a * 2.0 ** -24 * wide)
    for top in (1, groups // 2):
        same_choice(sonicmoe, logits, min(2, top * n), bias.flatten(), groups, top, 2, softmax)


def test_the_least_kept_group_need_not_be_the_one_in_doubt(sonicmoe):
    """Biases of 1e4 that cancel in one group alone, which ranks just ahead of or behind groups without any; also the two scores whose
    rounded sums stand the other way round than the sums."""
    bias = torch.tensor([1e4, -1e4, 0.0, 0, 0, 0, 0, 0])
    g = torch.Generator().manual_seed(1)
    logits = torch.randint(0, 64, (300, 8), generator=g) * 2.0 ** -14
    for top in (1, 2, 3):
        same_choice(sonicmoe, logits, 2, bias, 4, top, 2, False)
    s = torch.tensor([[0.5003, 0.5, 0.5001, 0.5]], dtype=torch.float64)
    x = torch.log(s / (1 - s)).float()
    same_choice(sonicmoe, x, 1, bias[:4], 2, 1, 2, False)


@pytest.mark.parametrize("E,groups", TABLES)
def test_a_group_of_nan_behind_one_of_the_lowest_logits(sonicmoe, E, groups):
    """Without a bias groups of one score rank by their logits, and NaN is below every number."""
    n = E // groups
    logits = torch.full((4, E), -math.inf)
    logits[0, :n], logits[0, 2 * n:3 * n] = math.nan, LOWEST
    logits[1, n:2 * n], logits[1, :n] = math.nan, LOWEST
    logits[2, :2 * n] = math.nan
    logits[3, -1], logits[3, 0] = LOWEST, math.nan
    for group_score in (1, 2):
        same_choice(sonicmoe, logits, 1, None, groups, 1, group_score, False)
