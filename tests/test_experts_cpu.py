"""CPU tests of the expert-layer operators' host side: the C entry points check
their arguments before any device work, and the operators refuse host tensors."""
import ctypes

import pytest
import torch

import efficient_linear_assignment_b200 as ela
from efficient_linear_assignment_b200 import _lib

NULL, ONE = ctypes.c_void_p(0), ctypes.c_void_p(256)
F32, F16, BF16, F64 = 0, 1, 2, 3


def test_host_tensors_are_refused():
    plan = ela.ExpertPlan(torch.zeros(2, dtype=torch.int32), torch.zeros(4, 1, dtype=torch.int32),
                          torch.zeros(4, dtype=torch.int32))
    x = torch.zeros(4, 8)
    for call in (lambda: ela.expert_plan(torch.zeros(4, dtype=torch.int64), 1), lambda: ela.expert_dispatch(x, plan),
                 lambda: ela.expert_combine(x, plan), lambda: ela.expert_linear(x.bfloat16(), torch.zeros(4, 8).bfloat16())):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_operators_are_registered():
    for name in ("expert_plan", "expert_dispatch", "expert_combine", "expert_linear"):
        assert hasattr(torch.ops.ela_native, name)


def test_plan_arguments():
    f = _lib.load().ela_expert_plan
    assert f(ONE, 2, 4, 4, ONE, ONE, ONE, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT  # id width
    assert f(ONE, 8, 4, 0, ONE, ONE, ONE, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT  # no experts
    assert f(ONE, 8, 4, 4097, ONE, ONE, ONE, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT
    assert f(ONE, 8, -1, 4, ONE, ONE, ONE, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT
    assert f(ONE, 8, 1 << 31, 4, ONE, ONE, ONE, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT
    assert f(NULL, 8, 4, 4, ONE, ONE, ONE, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT
    assert f(ONE, 8, 4, 4, NULL, ONE, ONE, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT


def test_dispatch_and_combine_arguments():
    lib = _lib.load()
    assert lib.ela_expert_dispatch(ONE, F64, 4, 1, 8, 8, ONE, ONE, 2, ONE, NULL) == _lib.ELA_ERR_ARGUMENT
    assert lib.ela_expert_dispatch(ONE, F32, 1 << 30, 4, 8, 8, ONE, ONE, 2, ONE, NULL) == _lib.ELA_ERR_ARGUMENT
    assert lib.ela_expert_dispatch(NULL, F32, 4, 1, 8, 8, ONE, ONE, 2, ONE, NULL) == _lib.ELA_ERR_ARGUMENT
    assert lib.ela_expert_dispatch(NULL, F32, 0, 1, 8, 8, NULL, NULL, 2, NULL, NULL) == _lib.ELA_OK  # nothing to do
    assert lib.ela_expert_combine(ONE, BF16, 4, 1, 8, 8, ONE, ONE, 2, ONE, F16, ONE, NULL) == _lib.ELA_ERR_ARGUMENT
    assert lib.ela_expert_combine(ONE, BF16, 4, 1, 8, 8, ONE, ONE, 0, ONE, F32, ONE, NULL) == _lib.ELA_ERR_ARGUMENT
    assert lib.ela_expert_combine(ONE, BF16, 4, 1, 8, 8, ONE, ONE, 2, ONE, F32, NULL, NULL) == _lib.ELA_ERR_ARGUMENT
    g = lib.ela_expert_combine_grad
    assert g(ONE, NULL, BF16, 4, 1, 8, 8, 8, ONE, ONE, 2, ONE, F32, NULL, ONE, NULL) == _lib.ELA_ERR_ARGUMENT  # dweights need y
    assert g(ONE, ONE, BF16, 4, 1, 8, 8, 8, ONE, ONE, 2, ONE, F16, ONE, NULL, NULL) == _lib.ELA_ERR_ARGUMENT
    assert g(ONE, ONE, BF16, 4, 1, 8, 8, 8, ONE, ONE, 2, ONE, F32, NULL, NULL, NULL) == _lib.ELA_OK  # nothing asked


def test_linear_arguments():
    lib = _lib.load()

    def forward(dtype=BF16, R=4, E=2, K=8, N=16, ldx=8, act=0, x=ONE, w=ONE, y=ONE, off=ONE, ldw=8):
        return lib.ela_expert_linear(x, w, NULL, NULL, off, dtype, R, E, K, N, ldx, 128, ldw, 16, act, y, NULL, NULL, 0, NULL)

    for bad in (dict(dtype=F32), dict(dtype=F64), dict(R=-1), dict(E=0), dict(E=4097), dict(K=0), dict(N=0), dict(act=4),
                dict(act=-1), dict(x=NULL), dict(w=NULL), dict(y=NULL), dict(off=NULL), dict(ldx=-8), dict(ldw=-1)):
        assert forward(**bad) == _lib.ELA_ERR_ARGUMENT, bad
    assert forward(R=0) == _lib.ELA_OK
    assert lib.ela_expert_linear_grad_input(NULL, ONE, ONE, BF16, 4, 2, 8, 16, 128, 8, ONE, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT
    assert lib.ela_expert_linear_grad_weight(ONE, ONE, ONE, BF16, 4, 2, 8, 16, 8, NULL, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT
    assert lib.ela_expert_linear_grad_act(ONE, NULL, ONE, BF16, 4, 2, 16, 2, ONE, NULL, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT
    assert lib.ela_expert_linear_grad_act(ONE, NULL, ONE, BF16, 4, 2, 16, 9, ONE, NULL, NULL, 0, NULL) == _lib.ELA_ERR_ARGUMENT
