"""CPU tests of the expert-layer operators' host side, with tensors that have no data."""
import ctypes
import glob
import os

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import efficient_linear_assignment_b200 as ela
from efficient_linear_assignment_b200 import _lib


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


def test_pointers_off_their_elements_are_refused():
    """The kernels would fault on them."""
    lib, null = _lib.load(), ctypes.c_void_p(0)
    f32, bf16, argument = 0, 2, _lib.ELA_ERR_ARGUMENT
    one, odd, half = ctypes.c_void_p(256), ctypes.c_void_p(257), ctypes.c_void_p(258)

    def each(f, pointers, *bad):
        """f with one of its pointers replaced, the others good."""
        for i in range(pointers):
            for p in bad:
                assert f(*[p if j == i else one for j in range(pointers)]) == argument, (i, p)

    each(lambda e, o, p, s: lib.ela_expert_plan(e, 8, 4, 4, o, p, s, null, 0, null), 4, odd, half)
    each(lambda x, p, o, r: lib.ela_expert_dispatch(x, f32, 4, 1, 8, 8, p, o, 2, r, null), 4, odd, half)
    each(lambda x, r: lib.ela_expert_dispatch(x, bf16, 4, 1, 8, 8, one, one, 2, r, null), 2, odd)
    each(lambda y, p, o, w, out: lib.ela_expert_combine(y, f32, 4, 1, 8, 8, p, o, 2, w, f32, out, null), 5, odd, half)
    each(lambda d, y, w, dy, dw: lib.ela_expert_combine_grad(d, y, f32, 4, 1, 8, 8, 8, one, one, 2, w, f32, dy, dw, null), 5, odd, half)
    each(lambda x, w, b, r, y, z: lib.ela_expert_linear(x, w, b, r, one, bf16, 4, 2, 8, 16, 8, 128, 8, 16, 0, y, z, null, 0, null), 6, odd)
    each(lambda o, z: lib.ela_expert_linear(one, one, null, null, o, bf16, 4, 2, 8, 16, 8, 128, 8, 16, 2, one, z, null, 0, null), 2, half)
    each(lambda dy, z, dz, db: lib.ela_expert_linear_grad_act(dy, z, one, bf16, 4, 2, 16, 1, dz, db, one, 1 << 20, null), 4, odd)
    each(lambda z, o, ws: lib.ela_expert_linear_grad_act(one, z, o, bf16, 4, 2, 16, 2, one, one, ws, 1 << 20, null), 3, half)
    each(lambda dz, w, o, dx: lib.ela_expert_linear_grad_input(dz, w, o, bf16, 4, 2, 8, 16, 128, 8, dx, null, 0, null), 4, odd)
    each(lambda dz, x, o, dw: lib.ela_expert_linear_grad_weight(dz, x, o, bf16, 4, 2, 8, 16, 8, dw, null, 0, null), 4, odd)
    # rows that TMA cannot read are copied into the workspace by 16-byte stores
    big = 1 << 24
    for ws in (odd, half, ctypes.c_void_p(264)):
        assert lib.ela_expert_linear(one, one, null, null, one, bf16, 400, 2, 9, 16, 9, 144, 9, 16, 0, one, null, ws, big, null) == argument
        assert lib.ela_expert_linear_grad_input(one, one, one, bf16, 4, 2, 9, 17, 153, 9, one, ws, big, null) == argument
        assert lib.ela_expert_linear_grad_weight(one, one, one, bf16, 4, 2, 9, 17, 9, one, ws, big, null) == argument
