"""GPU tests of expert_route's order where fp32 is short of digits.  Definitions and bounds are those
of test_expert_route_gpu.py."""
import pytest
import torch

from test_expert_route_gpu import check, gen

pytestmark = pytest.mark.gpu


def logit(s):
    return torch.log(s) - torch.log1p(-s)


def told_apart(a, b):
    """Rows whose pairs of keys are equal, or differ by more than 64-bit arithmetic is off by (an exponential
    of 60 by 60 * 2^-53 of itself)."""
    gap = (a - b).abs()
    return ((gap == 0) | (gap > 1e-12 * torch.maximum(a.abs(), b.abs()))).all(1)


@pytest.mark.parametrize("at", [-6.0, -9.0, -12.0, -20.0, -40.0, -60.0, -85.0])
@pytest.mark.parametrize("E,groups", [(16, 1), (64, 1), (256, 1), (256, 8), (1024, 1), (40, 5)])
def test_close_keys_of_small_sigmoids(at, E, groups):
    """A row without a large score, and biases no larger than the scores: the error of a sigmoid, as a part of it,
    grows with the logit, and pairs of keys lie within it."""
    T, g = 100, gen(E + int(-at))
    l = at + 0.3 * torch.randn(T, E, generator=g)
    bias = torch.zeros(E)
    bias[1::2] = 0.05 * torch.special.expit(torch.tensor(at - 1.0, dtype=torch.float64)).float()
    s = torch.special.expit(l[:, 0::2].double())
    l[:, 1::2] = logit((s - bias[1::2].double()).clamp(min=1e-45)).float()
    key = torch.special.expit(l.double()) + bias.double()
    gap = (key[:, 0::2] - key[:, 1::2]).abs() / key[:, 0::2]
    assert (gap < 2.0 ** -24 * max(8, -2 * at)).float().mean() > 0.5  # (the case is what it says)
    row = told_apart(key[:, 0::2], key[:, 1::2])
    k, kept = min(8, E // 2), max(1, groups // 2)
    check(l[row], k, "sigmoid", bias, groups, kept, "max")
    check(l[row], k, "sigmoid", bias, groups, kept, "top2" if groups > 1 else "max", renormalize=False)


@pytest.mark.parametrize("at", [-3.0, -9.0, -12.0, -20.0, -60.0])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups,kept", [(2, 1), (16, 5)])
def test_close_groups_of_small_sigmoids(at, biased, groups, kept):
    """Groups ranked by their two best scores, pairs of groups with nearly the same sum."""
    T, g = 400, gen(groups + int(-at))
    l = torch.full((T, groups, 4), at - 6.0)
    l[:, :, :2] = at + 0.2 * torch.randn(T, groups, 2, generator=g)
    s = torch.special.expit(l.double())
    x = (l[:, 0::2, 0] + 0.1).float()
    l[:, 1::2, 0] = x
    l[:, 1::2, 1] = logit(s[:, 0::2, 0] + s[:, 0::2, 1] - torch.special.expit(x.double())).float()
    total = torch.special.expit(l.double())[:, :, :2].sum(2)
    row = told_apart(total[:, 0::2], total[:, 1::2])
    assert row.float().mean() > 0.9
    l = l.flatten(1)[row]
    check(l, 4, "sigmoid", torch.zeros(l.shape[1]) if biased else None, groups, kept, "top2")


def test_sigmoids_below_the_normal_numbers():
    """Scores that an approximate reciprocal gives as 0, with biases as small."""
    g = gen(3)
    l = -87.0 - 4 * torch.rand(300, 32, generator=g)
    for bias in (torch.zeros(32), torch.randn(32, generator=g) * 2e-39, torch.randn(32, generator=g) * 1e-38):
        check(l, 6, "sigmoid", bias)
        check(l, 6, "sigmoid", bias, 4, 2, "top2")
    check(l, 6, "sigmoid", None, 4, 2, "top2")
