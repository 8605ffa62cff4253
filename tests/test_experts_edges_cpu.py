"""CPU tests of the expert-layer operators' host side, with tensors that have no data."""
import glob
import os

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import efficient_linear_assignment_b200 as ela


def fake_parts():
    bf = torch.bfloat16
    plan = ela.ExpertPlan(torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(4, 1, dtype=torch.int32, device="cuda"),
                          torch.empty(4, dtype=torch.int32, device="cuda"))
    x, w, g = torch.empty(4, 8, dtype=bf, device="cuda"), torch.empty(2, 16, 8, dtype=bf, device="cuda"), torch.empty(4, 1, device="cuda")
    b, r = torch.empty(2, 16, dtype=bf, device="cuda"), torch.empty(4, 16, dtype=bf, device="cuda")
    return [(lambda v: ela.expert_dispatch(v, plan), x), (lambda v: ela.expert_combine(v, plan, g), x),
            (lambda v: ela.expert_combine(x, plan, v), g), (lambda v: ela.expert_linear(v, w, offsets=plan.offsets), x),
            (lambda v: ela.expert_linear(x, v, offsets=plan.offsets), w),
            (lambda v: ela.expert_linear(x, w, v, offsets=plan.offsets), b),
            (lambda v: ela.expert_linear(x, w, None, v, offsets=plan.offsets), r)]


def test_forward_mode_is_refused():
    """A tangent is not dropped: forward-mode derivatives raise."""
    import torch.autograd.forward_ad as fwd
    with FakeTensorMode():
        for f, v in fake_parts():
            f(v)
            with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                f(fwd.make_dual(v, torch.empty_like(v)))


@pytest.mark.parametrize("shape", [(4,), (4, 1)])
def test_gradient_of_gates_has_their_shape(shape):
    """What a traced graph sees of the gradient of the weights, (T,) or (T, 1)."""
    with FakeTensorMode():
        y, w = torch.empty(4, 8, device="cuda", requires_grad=True), torch.empty(shape, device="cuda", requires_grad=True)
        plan = ela.ExpertPlan(torch.empty(3, dtype=torch.int32, device="cuda"),
                              torch.empty(4, 1, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int32, device="cuda"))
        dy, dw = torch.ops.ela_native.expert_combine_grad(torch.empty(4, 8, device="cuda"), y, plan.position, plan.offsets, w, True, True)
        assert dy.shape == y.shape and dw.shape == w.shape and dw.dtype == w.dtype


def test_kernels_that_start_early_read_coherently():
    """Every expert kernel may begin before the one that writes its inputs has ended; loads by
    the non-coherent path promise that nothing is written while the kernel lives."""
    root = os.path.dirname(os.path.abspath(ela.experts.__file__))
    files = glob.glob(os.path.join(root, "csrc", "ela_expert*.cu*"))
    assert len(files) >= 4
    for path in files:
        with open(path) as f:
            text = f.read()
        for word in ("__ldg", "ld.global.nc", "__restrict__"):
            assert word not in text, (path, word)
