"""GPU tests of the 4-bit experts where the kernels change their shape: many experts with many rows
each.  Definitions and bounds are those of test_expert_4bit_gpu.py."""
import pytest
import torch

import efficient_linear_assignment_b200 as ela
from test_expert_4bit_gpu import check, gen, product_case

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
