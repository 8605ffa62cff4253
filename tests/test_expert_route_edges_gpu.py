"""GPU tests of expert_route's order where fp32 is short of digits.  Definitions and bounds are those
of test_expert_route_gpu.py."""
import pytest
import torch

import efficient_linear_assignment_b200 as ela
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


def logits_and_masks(T, E, seed, value):
    """Usual logits and biases, a fifth of the experts closed by a large negative number."""
    g = gen(seed)
    bias = torch.randn(E, generator=g) * 0.1
    bias[::5] = value
    return torch.randn(T, E, generator=g) * 1.5, bias


@pytest.mark.parametrize("value", [-30.0, -1e4, -1e9, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masks_that_are_finite(value, score):
    """Experts closed by a finite bias: last in the order, and the others' order that of 64 bits."""
    for T, E, k, groups, kept in ((60, 256, 8, 8, 4), (60, 40, 6, 5, 2), (12, 1000, 8, 1, 1), (60, 20, 20, 1, 1)):
        l, bias = logits_and_masks(T, E, E, value)
        for by in ("max", "top2"):
            got = check(l, k, score, bias, groups, kept, by)
            assert k == E or (got.expert % 5 != 0).all()
    # close keys beside a mask
    l, bias = torch.randn(200, 12, generator=gen(2)), torch.zeros(12)
    bias[0], bias[2] = value, 0.01
    l[:, 2] = logit((torch.special.expit(l[:, 1].double()) - bias[2].double()).clamp(1e-3, 1)).float()
    s = torch.special.expit(l.double()) + bias.double()
    row = told_apart(s[:, 1:2], s[:, 2:3])
    check(l[row], 4, "sigmoid", bias)
    check(l[row], 3, "sigmoid", bias, 4, 2, "max")


def time_of(call, passes=10):
    for _ in range(3):
        call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(passes):
            call()
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("T,E,groups,kept", [(8192, 256, 8, 4), (8192, 256, 1, 1), (1024, 4096, 1, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_a_finite_mask_costs_what_others_do(T, E, groups, kept, score):
    """(The same takes as long; where every key was in doubt it took 7 to 300 times as long.)"""
    times = []
    for value in (0.0, -1e9):
        l, bias = (v.cuda() for v in logits_and_masks(T, E, 5, value))
        times.append(time_of(lambda: ela.expert_route(l, 8, score, bias, groups, kept, "top2" if groups > 1 else "max")))
    assert times[1] < 3 * times[0], times


def test_sums_of_groups_past_fp32s_range():
    """Two biases whose sum is an infinity in fp32: in order among themselves, and not as closed groups are."""
    inf, big = float("inf"), 3e38
    l = torch.randn(6, 16, generator=gen(4))
    for bias in ([2e38, 2e38, 0, 0, 3e38, 2e38, 0, 0, 2.5e38, 2e38, 0, 0, 0, 0, 0, 0], [-big] * 4 + [-2.9e38] * 4 + [-2.8e38] * 4 + [-3.1e38] * 4,
                 [0, -inf, -inf, -inf] + [-big] * 4 + [-inf] * 4 + [-2.9e38] * 4, [big, -big, 0, 0] * 2 + [-big, -big, big, 1] * 2,
                 [-inf] * 4 + [1, -inf, -inf, -inf] + [-big] * 4 + [-inf] * 4):
        for score in ("softmax", "sigmoid"):
            for kept in (1, 2, 3):
                check(l, 2, score, torch.tensor(bias), 4, kept, "top2")


@pytest.mark.parametrize("E,k,groups,kept", [(256, 8, 1, 1), (256, 8, 8, 4), (1000, 64, 1, 1), (4096, 8, 1, 1), (4096, 20, 16, 3), (512, 64, 1, 1), (300, 1, 1, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_many_equal_keys(E, k, groups, kept, score):
    """Rows with more equal experts than are ranked: zeros, two and three values, some closed, a few above the rest."""
    g = gen(E + k)
    l = torch.zeros(9, E)
    l[1] = -4.0
    l[2, E // 2:] = 1.0
    l[3] = torch.randint(0, 3, (E,), generator=g).float()
    l[4, torch.randperm(E, generator=g)[:3]] = 2.0
    l[5, torch.rand(E, generator=g) < 0.5] = -float("inf")
    l[6, :5] = -float("inf")
    l[7] = torch.where(torch.rand(E, generator=g) < 0.5, 0.0, -0.0)
    l[8, -1] = 3.0
    coarse = torch.randint(0, 2, (E,), generator=g) * 0.25
    for bias in (None, torch.zeros(E), torch.full((E,), 0.3), coarse):
        for by in ("max", "top2"):
            for dtype in (torch.float32, torch.bfloat16):
                check(l.to(dtype), k, score, bias, groups, kept, by)
    # equal logits but for one that is larger by less than fp32 tells behind them, with a bias
    s = torch.special.expit(torch.tensor(0.3, dtype=torch.float64))
    l, bias = torch.full((2, E), 0.3), torch.zeros(E)
    bias[E - 2] = 0.02
    for t, d in enumerate((1e-9, -1e-9)):
        l[t, E - 2] = logit(s + d - bias[E - 2].double()).float()
    check(l, k, "sigmoid", bias)
    # not a number: all of a softmax's keys, and some of a sigmoid's
    l = torch.zeros(2, E).cuda()
    l[0, 7] = float("nan")
    got = ela.expert_route(l, k, score, torch.zeros(E, device="cuda"))
    first = list(range(k)) if score == "softmax" else [7] + [e for e in range(k) if e != 7][:k - 1]
    assert got.expert[0].tolist() == first and got.expert[1].tolist() == list(range(k))


@pytest.mark.parametrize("T,E,groups,kept", [(8192, 256, 8, 4), (8192, 256, 1, 1), (1024, 4096, 1, 1)])
@pytest.mark.parametrize("biased", [True, False])
def test_equal_keys_cost_what_others_do(T, E, groups, kept, biased):
    """(Rows of zeros took 8 to 280 times as long; now 2 to 4.5 times, the most where groups tie and 64 bits tell so.)"""
    times = []
    for spread in (1.5, 0.0):
        l = (torch.randn(T, E, generator=gen(5)) * spread).cuda()
        times.append(time_of(lambda: ela.expert_route(l, 8, "sigmoid", torch.zeros(E, device="cuda") if biased else None, groups, kept, "top2" if groups > 1 else "max")))
    assert times[1] < 6 * times[0], times


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_with_one_open_expert(score):
    """By the sum of two such a group ranks with the closed ones, by index, and after every group with two."""
    no = -float("inf")
    l = torch.tensor([[no, no, 5.0, no, no, no], [no, no, 5.0, no, -3.0, -4.0], [5.0, no, 1.0, no, 2.0, no], [no, no, no, no, no, 1.0]])
    for bias in (None, torch.zeros(6)):
        top2 = check(l, 2, score, bias, 3, 1, "top2").expert.tolist()
        assert top2 == [[-1, -1], [4, 5], [0, -1], [-1, -1]]
        most = check(l, 2, score, bias, 3, 1, "max").expert.tolist()
        assert most == [[2, -1], [2, -1], [0, -1], [5, -1]]
        assert check(l, 2, score, bias, 3, 2, "top2").expert.tolist() == [[2, -1], [4, 5], [0, 2], [-1, -1]]


@pytest.mark.parametrize("E", [30, 64, 100, 193, 200, 230, 256, 320, 512])
@pytest.mark.parametrize("k", [9, 17, 33, 40, 64])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_many_choices(E, k, score):
    """More choices than a row's threads have largest keys, two each: usual rows, and rows with many equal keys."""
    k = min(k, E)
    g = gen(E + k)
    l = torch.randn(20, E, generator=g) * 1.5
    l[10:] = l[10:].round()
    l[18], l[19] = 0.0, (torch.arange(E) % 2).float()
    for bias in (None, torch.zeros(E), torch.randn(E, generator=g) * 0.1):
        check(l, k, score, bias)
        if E % 2 == 0 and k <= E // 2:
            check(l, k, score, bias, 2, 1, "top2")


def test_the_gradient_operator_checks_its_arguments():
    l, dw = torch.zeros(5, 8, device="cuda"), torch.ones(5, 3, device="cuda")
    expert = ela.expert_route(l, 3).expert
    grad = torch.ops.ela_native.expert_route_grad
    want = grad(dw, l, expert, 0, False, 1.0)
    assert torch.equal(grad(dw.t().contiguous().t(), l, expert.t().contiguous().t(), 0, False, 1.0), want)
    for bad in ((dw[:4], l, expert), (dw, l, expert[:4]), (dw[:, :2], l, expert), (dw, l[:4], expert), (dw, l[0], expert), (dw[0], l, expert[0]),
                (dw.cpu(), l, expert), (dw, l, expert.cpu())):
        with pytest.raises(ValueError):
            grad(*bad, 0, False, 1.0)
    for bad in ((dw.double(), l, expert), (dw, l, expert.long()), (dw, l.double(), expert)):
        with pytest.raises(TypeError):
            grad(*bad, 0, False, 1.0)
