"""GPU tests of the 4-bit experts at the edges: many experts with many rows each, where the tiles change
their shape, and activations far out.  Definitions and bounds are those of test_expert_4bit_gpu.py."""
import math

import pytest
import torch

import efficient_linear_assignment_b200 as ela
from test_expert_4bit_gpu import act64, check, gen, product_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,share,K,N", [(513, 128, 384, 264), (600, 128, 1000, 264), (1024, 128, 1024, 256), (1537, 125, 520, 64), (2048, 120, 648, 72),
                                         (2561, 128, 384, 40), (3585, 128, 384, 40), (4096, 128, 256, 24)])
@pytest.mark.parametrize("skewed", [False, True])
def test_wide_tiles_of_many_experts(E, share, K, N, skewed):
    """Tables of experts that leave room for few stages, three to eight blocks of 128 inputs: the sums, and the
    same bits every time."""
    g, R = gen(E), E * share
    if skewed:  # some with thousands of rows, a tenth with none
        share_of = torch.rand(E, generator=g) ** 4 * (torch.rand(E, generator=g) < 0.9)
        counts = torch.multinomial(share_of, R - 70, replacement=True, generator=g).bincount(minlength=E).tolist()
        first = 30
    else:
        counts, first = [share] * E, 0
    x, w, _, _, off = product_case(R, E, K, N, torch.bfloat16, E, counts, first, bias=False, residual=False, group=64)
    y = check(x, w, None, None, off, "none")
    dx, o = x.cuda(), torch.tensor(off, dtype=torch.int32, device="cuda")
    for _ in range(5):
        assert torch.equal(ela.expert_linear_4bit(dx, w, offsets=o), y)
    ela.expert_check()


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_activations_far_out(act):
    """The tails themselves, by a bound that shrinks with them, and every row the same.

    Sums are exact here (one product each).  GELU: the polynomial of erfc is off by 5 % of a tail up to 14
    (computed in 64 bits) and by 7.5e-8 of it halved, its evaluation by 16 steps of 2^-24 of the Gaussian.  SiLU: the
    exponent's rounding, 2.4 |z| 2^-24, the exponential, the sum and the division.  A tail below 2^-126 may come out
    as 0, so a result below |z| 2^-126.  Rounded to bf16 once."""
    K, N = 64, 48
    w = ela.expert_quantize(torch.eye(N, K).to(torch.bfloat16).mul(7).cuda(), 32)
    z = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 1e-4, -1e-4, 0.5, -0.5, 1.0, -1.0, 2.0, -2.0, 3.0, -3.0, 4.0, -4.0, 5.0, -5.0, 6.0, -6.0, 7.0, -7.0, 8.0, -8.0,
                      10.0, -10.0, 12.0, -12.0, 13.0, -13.0, 20.0, -20.0, 40.0, -40.0, 60.0, -60.0, 80.0, -80.0, 86.0, -86.0, 89.0, -89.0, 100.0, -100.0,
                      1e18, -1e18, 3e37, -3e37])
    x = torch.zeros(300, K)
    x[:, :N] = z / 7
    x = x.to(torch.bfloat16).cuda()
    s = (x[0, :N].double() * 7).cpu()
    want = act64(s, act)
    a = s.abs()
    if act == "gelu":
        tail, gauss = 0.5 * torch.special.erfc(a / math.sqrt(2)), torch.exp(-s * s / 2)
        own = a * (torch.minimum(0.05 * tail, torch.full_like(a, 7.5e-8)) + 16 * 2.0 ** -24 * gauss + 2.0 ** -126) + 2.0 ** -22 * want.abs()
    else:
        own = a * 2.0 ** -126 + (2.4 * a.clamp(max=100) + 16) * 2.0 ** -24 * want.abs() if act == "silu" else torch.zeros_like(s)
    for rows in (2, 300):
        y = ela.expert_linear_4bit(x[:rows], w, None, None, act)
        assert y.isfinite().all() and (y == y[0]).all()
        off = (y[0].double().cpu() - want).abs()
        worst = (off - own - 2.0 ** -8 * 1.01 * want.abs() - 2.0 ** -133).max().item()
        assert worst <= 0, (worst, y[0], want)
