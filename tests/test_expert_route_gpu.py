"""GPU tests of expert_route against its definition in 64 bits.

Bounds.  In fp32 an exponent's rounding moves its exponential by spread * 2^-24 (spread:
the largest difference of logits that is formed), the exponential and the division are off
by 2^-22 and 2^-24, and a row's sum by at most 29 additions one after the other, 2^-24
each: a weight is off by at most (48 + spread) * 2^-24 of itself.  The gradient is a
difference of such products, each off by twice that and the k additions of the mean, and
is rounded once to the logits' type.  Results below 2^-126 may come out as 0.
"""
import math

import pytest
import torch

import efficient_linear_assignment_b200 as ela

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -126}
LOW = -math.inf


def gen(seed):
    return torch.Generator().manual_seed(seed)


def by_size(values):
    """Places from the largest value on, NaN first, equal ones in order."""
    return sorted(range(len(values)), key=lambda i: (0 if values[i] != values[i] else 1, -values[i] if values[i] == values[i] else 0, i))


def scores(row, score):
    l = row.double()
    if score == "sigmoid":
        return torch.special.expit(l)
    return torch.softmax(l, 0) if not torch.isneginf(l).all() else torch.zeros_like(l)


def choice_by_definition(row, k, score, bias, groups, kept, by):
    """One row's experts, the straightforward way."""
    E = len(row)
    s = scores(row, score)
    key = row.double() if bias is None else s + bias.double()
    value = s if bias is None else key
    out = torch.isneginf(row) | (torch.isneginf(bias) if bias is not None else False)
    key, value = key.masked_fill(out, LOW).tolist(), value.masked_fill(out, LOW).tolist()
    if kept < groups:
        S = E // groups
        rank = []
        for g in range(groups):
            part = (key if by == "max" else value)[g * S:(g + 1) * S]
            top = [part[i] for i in by_size(part)]
            rank.append(top[0] if by == "max" else top[0] + top[1])
        for g in by_size(rank)[kept:]:
            key[g * S:(g + 1) * S] = [LOW] * S
    return [e if key[e] != LOW else -1 for e in by_size(key)[:k]]


def weights_by_definition(l, at, score, renormalize, scale):
    """(T, k) weights of the chosen experts, 64 bits, differentiable in l."""
    gone = at < 0
    logs = torch.nn.functional.logsigmoid(l) if score == "sigmoid" else torch.log_softmax(l, 1)
    mine = logs.gather(1, at.clamp(min=0))
    if renormalize:
        mine = torch.where(gone.all(1, keepdim=True), torch.zeros_like(mine), mine.masked_fill(gone, LOW))
        w = torch.softmax(mine, 1)
    else:
        w = torch.exp(mine)
    return (scale * w).masked_fill(gone, 0.0)


def check(logits, k, score="softmax", bias=None, groups=1, kept=None, by="max", renormalize=True, scale=1.0, seed=0):
    T, E = logits.shape
    kept = groups if kept is None else kept
    dl = logits.detach().cuda().requires_grad_()
    got = ela.expert_route(dl, k, score, None if bias is None else bias.cuda(), groups, kept, by, renormalize, scale)
    assert got.expert.dtype == torch.int32 and got.weights.dtype == torch.float32 and got.expert.shape == got.weights.shape == (T, k)
    quiet = ela.expert_route(dl.detach(), k, score, None if bias is None else bias.cuda(), groups, kept, by, renormalize, scale)
    assert torch.equal(quiet.expert, got.expert) and torch.equal(quiet.weights, got.weights.detach())
    want = torch.tensor([choice_by_definition(logits[t], k, score, bias, groups, kept, by) for t in range(T)]).view(T, k)
    assert torch.equal(got.expert.cpu().long(), want)
    # rows without any expert stay out of the 64-bit graph (their softmax is 0 / 0)
    some = ~torch.isneginf(logits).all(1)
    l = logits[some].double().requires_grad_()
    ref = weights_by_definition(l, want[some], score, renormalize, scale)
    w = got.weights.detach().cpu().double()
    assert (w[~some] == 0).all() and (got.weights.detach().cpu()[want < 0] == 0).all()
    lf = logits[some].double().masked_fill(torch.isneginf(logits[some]), 0.0)
    picked = lf.gather(1, want[some].clamp(min=0))
    most = lf.masked_fill(torch.isneginf(logits[some]), LOW).amax(1, keepdim=True) if not renormalize else picked.amax(1, keepdim=True)
    spread = (most - picked).abs().clamp(max=200) if score == "softmax" or renormalize else torch.zeros_like(picked)
    rel = (48 + spread) * 2.0 ** -24
    off = (w[some] - ref.detach()).abs()
    assert (off <= rel * ref.detach().abs() + 2.0 ** -126 * abs(scale)).all(), off.max()
    # gradient
    dw = torch.randn(T, k, generator=gen(seed + 1))
    (d,) = torch.autograd.grad(got.weights, dl, dw.cuda())
    assert d.dtype == logits.dtype and d.shape == logits.shape
    dref = torch.autograd.grad(ref, l, dw[some].double())[0]
    dref = torch.nan_to_num(dref, nan=0.0)  # (experts that are closed: the log of 0 in a graph that does not use it)
    d = d.cpu().double()
    assert (d[~some] == 0).all()
    p = torch.softmax(l.detach(), 1) if score == "softmax" and not renormalize else torch.zeros_like(dref).scatter_add(
        1, want[some].clamp(min=0), ref.detach().abs() / abs(scale) * (want[some] >= 0))
    c = torch.zeros_like(dref).scatter_add(1, want[some].clamp(min=0), (dw[some].double() * scale).abs() * (want[some] >= 0))
    mean = (dw[some].double() * ref.detach()).abs().sum(1, keepdim=True)
    err = (2 * (48 + spread.amax(1, keepdim=True).clamp(max=100)) + k + 8) * 2.0 ** -24 * p * (c + mean)
    if score == "softmax" and not renormalize:  # every expert's exponent
        wide = (l.detach().masked_fill(torch.isneginf(l.detach()), 0.0) - most).abs().clamp(max=200)
        err = err + wide * 2.0 ** -24 * p * (c + mean)
    # The 64-bit gradient's own error: an expert that is not chosen gets p_i * sum_j dlog_j, which is 0 in the
    # formula and the rounding of k terms here, (k + 4) * 2^-53 of their magnitudes, c_j w_j and its mean's each.
    err = err + (k + 4) * 2.0 ** -52 * mean
    bound = err + 1.01 * U[logits.dtype] * (dref.abs() + err) + TINY[logits.dtype] * (1 + c + mean)
    worst = ((d[some] - dref).abs() - bound).max().item() if dref.numel() else -1
    assert worst <= 0, worst
    return got


def make(T, E, dtype, seed, masked=0.0, padding=0, spread=1.5):
    g = gen(seed)
    l = torch.randn(T, E, generator=g) * spread
    if masked:
        l = l.masked_fill(torch.rand(T, E, generator=g) < masked, LOW)
    if padding:
        l[T - padding:] = LOW
    return l.to(dtype)


SIZES = [(1, 1, 1), (1, 2, 1), (8, 16, 2), (5, 7, 3), (129, 8, 8), (131, 9, 2), (33, 33, 4), (70, 64, 6), (37, 100, 8), (64, 128, 8), (21, 160, 6),
         (40, 256, 8), (9, 257, 16), (6, 512, 64), (5, 513, 7), (4, 1000, 9), (3, 4096, 64)]


@pytest.mark.parametrize("T,E,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_sizes(T, E, k, dtype, score):
    for renormalize in (True, False):
        check(make(T, E, dtype, T + E), k, score, renormalize=renormalize, seed=E)
        check(make(T, E, dtype, T + E + 1, masked=0.3, padding=T // 3), k, score, bias=torch.randn(E, generator=gen(E)) * 0.2,
              renormalize=renormalize, scale=2.5, seed=E + 7)


@pytest.mark.parametrize("E,groups,kept,k", [(8, 2, 1, 4), (16, 8, 3, 5), (12, 3, 2, 8), (64, 8, 4, 6), (256, 8, 4, 8), (160, 8, 3, 6), (30, 15, 4, 7),
                                             (256, 128, 5, 10), (6, 6, 3, 3), (512, 16, 4, 8), (768, 4, 2, 16), (2048, 64, 8, 8), (90, 9, 9, 4)])
@pytest.mark.parametrize("by", ["max", "top2"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups(E, groups, kept, k, by, score):
    if by == "top2" and E == groups:
        return
    for dtype, biased, masked in ((torch.float32, True, 0.0), (torch.bfloat16, False, 0.0), (torch.float32, False, 0.6), (torch.bfloat16, True, 0.4)):
        bias = torch.randn(E, generator=gen(3 * E)) * 0.1 if biased else None
        check(make(24, E, dtype, E + k, masked=masked, padding=2), k, score, bias, groups, kept, by, renormalize=biased, seed=k)


def test_ties_go_to_the_lowest_index():
    l = torch.zeros(4, 40)
    l[1, ::2] = 1.0
    l[2, 35:] = 2.0
    l[3] = -1.0
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(40)):
            for dtype in (torch.float32, torch.bfloat16):
                got = check(l.to(dtype), 6, score, bias)
                assert got.expert[0].tolist() == [0, 1, 2, 3, 4, 5] and got.expert[1].tolist() == [0, 2, 4, 6, 8, 10]
                assert got.expert[2].tolist() == [35, 36, 37, 38, 39, 0]
        got = check(l, 4, score, None, 10, 2, "top2")
        assert got.expert[0].tolist() == [0, 1, 2, 3]
    zeros = torch.tensor([[0.0, -0.0, 0.0, -0.0]])
    assert ela.expert_route(zeros.cuda(), 4).expert.tolist() == [[0, 1, 2, 3]]
    # coarse logits, many equal ones in every row
    check((make(200, 256, torch.float32, 5) * 2).round().div(2), 8, "sigmoid", torch.zeros(256))
    check((make(200, 64, torch.float32, 6) * 2).round().div(2), 8, "softmax", (torch.randn(64, generator=gen(1))).round() / 4)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups", [(16, 1), (64, 1), (256, 1), (256, 8), (1024, 1), (40, 5)])
def test_keys_closer_than_32_bits_tell(score, E, groups):
    """Biases that bring pairs of keys within rounding of each other: the order is that of 64 bits."""
    T = 64
    g = gen(E)
    l = torch.randn(T, E, generator=g)
    bias = torch.zeros(E)
    s = torch.softmax(l.double(), 1) if score == "softmax" else torch.special.expit(l.double())
    # sigmoid: the second of a pair gets the logit whose score lies next to the first's with another bias
    bias[1::2] = 0.01
    if score == "sigmoid":
        want = (s[:, 0::2] - bias[1::2].double()).clamp(1e-3, 1 - 1e-3)
        l[:, 1::2] = torch.log(want / (1 - want)).float()
    else:  # softmax: a pair's logits a few units of the last place apart, without a bias between them
        bias[:] = torch.arange(E // 2).repeat_interleave(2) * 1e-4
        l[:, 1::2] = l[:, 0::2] * (1 + 2.0 ** -22)
    s = torch.softmax(l.double(), 1) if score == "softmax" else torch.special.expit(l.double())
    key = s + bias.double()
    gaps = (key[:, 0::2] - key[:, 1::2]).abs()
    close = (gaps < 2.0 ** -22 * key[:, 0::2].abs()) & (gaps > 1e-14)
    assert close.float().mean() > 0.3  # (the case is what it says)
    row = gaps.masked_fill(gaps == 0, 1.0).amin(1) > 1e-14  # 64 bits tell
    check(l[row], min(8, E // 2), score, bias, groups, max(1, groups // 2), "max")
    check(l[row], min(8, E // 2), score, bias, groups, max(1, groups // 2), "top2" if groups > 1 else "max", renormalize=False)
    if score == "softmax":
        check(l[row], min(8, E // 2), score, None, groups, max(1, groups // 2), "top2" if groups > 1 else "max")


def test_a_close_key_behind_an_equal_one():
    """The last choice, an equal logit behind it, and one that is larger by less than fp32 tells."""
    s = 1 / (1 + math.exp(-0.3))
    for d in (1e-9, -1e-9):
        b = torch.tensor([0.0, 0.0, 0.02, -3.0])
        want = s + d - b[2].double().item()
        l = torch.tensor([[0.3, 0.3, math.log(want / (1 - want)), 4.0]], dtype=torch.float32)
        check(l, 1, "sigmoid", b)
        check(l, 2, "sigmoid", b)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masks(score):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        lowest = torch.finfo(dtype).min
        l = make(6, 24, dtype, 3)
        l[0] = LOW                       # nothing left
        l[1, 1:] = LOW                   # one left
        l[2, :22] = LOW                  # two left
        l[3] = lowest                    # masked by the type's lowest value, all
        l[4, 3:] = lowest                # and all but three
        for renormalize in (True, False):
            got = check(l, 4, score, None, renormalize=renormalize)
            assert got.expert[0].tolist() == [-1] * 4 and got.expert[1].tolist() == [0, -1, -1, -1]
            assert got.expert[3].tolist() == [0, 1, 2, 3]
            if renormalize:
                assert torch.allclose(got.weights[3].detach(), torch.full((4,), 0.25, device="cuda"), rtol=1e-6, atol=0)
        bias = torch.zeros(24)
        bias[::2] = LOW  # experts closed to every token
        got = check(l, 4, score, bias)
        assert (got.expert[got.expert >= 0] % 2 == 1).all() and got.expert[1].tolist() == [-1] * 4


def test_infinities_and_nan():
    l = make(5, 20, torch.float32, 9)
    l[0, 7] = math.inf
    l[1, 3] = math.nan
    l[2, 19] = -math.nan
    l[3, 2] = l[3, 9] = math.nan
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(20)):
            got = ela.expert_route(l.cuda(), 3, score, None if bias is None else bias.cuda())
            assert ((got.expert >= 0) & (got.expert < 20)).all()
            if bias is None or score == "sigmoid":
                assert got.expert[0, 0] == 7 and got.expert[1, 0] == 3 and got.expert[2, 0] == 19
                assert got.expert[3, :2].tolist() == [2, 9]
            assert got.weights[1:4].isnan().any(1).all() and got.weights[4].isfinite().all()
    assert ela.expert_route(l[:1].cuda(), 2, "sigmoid", renormalize=False).weights[0, 0] == 1.0


def test_small_and_large_scores_have_ratios():
    l = torch.tensor([[-300.0, -301.0, -302.0, -310.0], [300.0, 299.0, -300.0, 0.0], [-3e38, -2e38, -3e38, -3e38]])
    for score in ("softmax", "sigmoid"):
        check(l, 2, score)
        check(l, 4, score, renormalize=False)


def test_gradient_against_differences():
    h = 1e-4
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            l = make(3, 12, torch.float32, 4)
            dl = l.cuda().requires_grad_()
            got = ela.expert_route(dl, 3, score, renormalize=renormalize, scale=1.5)
            dw = torch.randn(3, 3, generator=gen(8))
            (d,) = torch.autograd.grad(got.weights, dl, dw.cuda())
            at = got.expert.cpu().long()
            for t in range(3):
                for e in range(12):
                    up, down = l.double(), l.double()
                    up[t, e] += h
                    down[t, e] -= h
                    q = [(weights_by_definition(v, at, score, renormalize, 1.5) * dw.double()).sum() for v in (up, down)]
                    # the quotient is off by h^2 / 6 of a third derivative (under 4 * 1.5 * 3 dw's) and cancellation
                    assert abs((q[0] - q[1]) / (2 * h) - d[t, e].item()) <= 1e-6 + 1e-6 * dw.abs().max()


def test_gradient_of_one_renormalized_choice_is_zero():
    """The weight of a single choice is the scale, whatever the logits."""
    for score in ("softmax", "sigmoid"):
        l = make(300, 216, torch.float32, 5, padding=4).cuda().requires_grad_()
        w = ela.expert_route(l, 1, score, scale=2.5).weights
        assert (w[:296] == 2.5).all() and (w[296:] == 0).all()
        (d,) = torch.autograd.grad(w, l, torch.randn(300, 1, generator=gen(6)).cuda() * 5)
        assert (d == 0).all()


def test_strides_broadcast_gradients_and_offsets():
    wide = make(50, 64, torch.bfloat16, 11)
    for view in (wide[:, :31], wide[:, 1:33], wide[::2, :32], wide[:, ::2], wide.t()):
        check(view, 3)
        check(view, 3, "sigmoid", torch.randn(view.shape[1], generator=gen(2)) * 0.1, renormalize=False)
    dl = wide.float().cuda().requires_grad_()
    w = ela.expert_route(dl, 4, renormalize=False).weights
    (a,) = torch.autograd.grad(w.sum(), dl, retain_graph=True)  # an expanded gradient
    (b,) = torch.autograd.grad(w, dl, torch.ones(50, 4, device="cuda"))
    assert torch.equal(a, b)
    one = wide[:1].float().cuda().expand(50, 64).requires_grad_()  # rows that are one row
    out = ela.expert_route(one, 4)
    assert (out.expert == out.expert[0]).all()
    # rows far apart: offsets past 32 bits
    rows = torch.as_strided(torch.zeros(2 ** 32 + 128, dtype=torch.bfloat16, device="cuda"), (3, 64), (2 ** 31, 1))
    rows.copy_(wide[:3])
    got = ela.expert_route(rows, 4)
    want = ela.expert_route(wide[:3].cuda(), 4)
    assert torch.equal(got.expert, want.expert) and torch.equal(got.weights, want.weights)


def test_no_rows():
    for E in (4, 600):
        l = torch.zeros(0, E, device="cuda", requires_grad=True)
        got = ela.expert_route(l, 2)
        assert got.expert.shape == (0, 2) and torch.autograd.grad(got.weights.sum(), l)[0].shape == (0, E)


def test_same_bits_on_any_stream_and_in_a_graph():
    l = make(3000, 96, torch.float32, 13).cuda()
    bias = (torch.randn(96, generator=gen(3)) * 0.1).cuda()
    call = lambda: ela.expert_route(l, 6, "sigmoid", bias, 8, 3, "top2", True, 2.0)  # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = call()
    l.copy_(make(3000, 96, torch.float32, 14))
    graph.replay()
    fresh = call()
    assert all(torch.equal(a, b) for a, b in zip(fresh, third)) and not torch.equal(first.expert, third.expert)


def test_training_step_in_a_graph():
    l = make(100, 32, torch.float32, 15).cuda().requires_grad_()
    dw = torch.randn(100, 2, device="cuda")

    def step():
        return torch.autograd.grad(ela.expert_route(l, 2, renormalize=False).weights, l, dw)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert torch.equal(got, want)


def test_refusals():
    l = torch.zeros(4, 12, device="cuda")
    ok = dict(k=2)
    for bad in (dict(k=0), dict(k=13), dict(k=2, groups=5), dict(k=2, groups=0), dict(k=2, groups=3, groups_kept=4), dict(k=2, groups=3, groups_kept=0),
                dict(k=5, groups=3, groups_kept=1), dict(k=2, score="relu"), dict(k=2, group_score="top3"), dict(k=2, groups=12, groups_kept=6, group_score="top2"),
                dict(k=2, scale=math.inf), dict(k=2, scale=math.nan), dict(k=2, bias=torch.zeros(11, device="cuda")), dict(k=2, bias=torch.zeros(12)),
                dict(k=2, bias=torch.zeros(1, 12, device="cuda"))):
        with pytest.raises(ValueError):
            ela.expert_route(l, **bad)
    with pytest.raises(ValueError):
        ela.expert_route(torch.zeros(4, 100, device="cuda"), 65)
    with pytest.raises(ValueError):
        ela.expert_route(torch.zeros(4, 4097, device="cuda"), 2)
    with pytest.raises(ValueError):
        ela.expert_route(torch.zeros(12, device="cuda"), **ok)
    with pytest.raises(TypeError):
        ela.expert_route(l.double(), **ok)
    with pytest.raises(TypeError):
        ela.expert_route(l, 2, bias=torch.zeros(12, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="CUDA"):
        ela.expert_route(l.cpu(), **ok)
    leaf = l.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ela.expert_route(leaf, 2).weights.sum(), leaf, create_graph=True)
