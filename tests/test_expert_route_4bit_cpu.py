"""CPU tests of the routing and 4-bit operators' host side: the C entry points check their
arguments before any device work, the operators refuse host tensors and lost gradients."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import efficient_linear_assignment_b200 as ela
from efficient_linear_assignment_b200 import _lib

NULL, ONE, HALF, ODD = ctypes.c_void_p(0), ctypes.c_void_p(256), ctypes.c_void_p(258), ctypes.c_void_p(257)
F32, F16, BF16, F64 = 0, 1, 2, 3
ARGUMENT = _lib.ELA_ERR_ARGUMENT


def test_host_tensors_are_refused():
    w = torch.zeros(4, 64).bfloat16()
    q = ela.Expert4Bit(torch.zeros(4, 8, dtype=torch.int32), torch.zeros(1, 4).bfloat16(), 64, 64)
    for call in (lambda: ela.expert_route(torch.zeros(4, 8), 2), lambda: ela.expert_quantize(w), lambda: ela.expert_dequantize(q),
                 lambda: ela.expert_linear_4bit(torch.zeros(2, 64).bfloat16(), q)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_names_are_checked():
    for bad in (dict(score="tanh"), dict(group_score="mean")):
        with pytest.raises(ValueError, match="Options"):
            ela.expert_route(torch.zeros(4, 8), 2, **bad)


def test_route_arguments():
    lib = _lib.load()

    def route(logits=ONE, dtype=F32, T=4, E=12, ld=12, k=2, score=0, bias=NULL, groups=1, kept=1, by=0, scale=1.0, expert=ONE, weights=ONE):
        return lib.ela_expert_route(logits, dtype, T, E, ld, k, score, bias, groups, kept, by, 1, scale, expert, weights, NULL)

    for bad in (dict(dtype=F64), dict(T=-1), dict(E=0), dict(E=4097), dict(ld=-1), dict(k=0), dict(k=13), dict(E=100, k=65), dict(score=2), dict(score=-1),
                dict(groups=0), dict(groups=5), dict(groups=3, kept=0), dict(groups=3, kept=4), dict(groups=3, kept=1, k=5), dict(by=2),
                dict(groups=12, kept=2, by=1), dict(scale=float("inf")), dict(scale=float("nan")), dict(T=1 << 30, k=2), dict(T=1 << 31, k=1),
                dict(logits=NULL), dict(expert=NULL), dict(weights=NULL), dict(logits=HALF), dict(bias=HALF), dict(expert=ODD), dict(weights=HALF),
                dict(dtype=BF16, logits=ODD)):
        assert route(**bad) == ARGUMENT, bad
    assert route(T=0, logits=NULL, expert=NULL, weights=NULL) == _lib.ELA_OK

    def grad(logits=ONE, dtype=F32, T=4, E=12, ld=12, k=2, score=0, scale=1.0, expert=ONE, dw=ONE, dl=ONE):
        return lib.ela_expert_route_grad(logits, dtype, T, E, ld, k, score, 0, scale, expert, dw, dl, NULL)

    for bad in (dict(dtype=F64), dict(T=-1), dict(E=0), dict(k=0), dict(k=13), dict(score=2), dict(scale=float("nan")), dict(logits=NULL), dict(expert=NULL),
                dict(dw=NULL), dict(dl=NULL), dict(logits=HALF), dict(expert=HALF), dict(dw=HALF), dict(dl=HALF), dict(dtype=F16, dl=ODD)):
        assert grad(**bad) == ARGUMENT, bad
    assert grad(T=0, logits=NULL) == _lib.ELA_OK


def test_4bit_arguments():
    lib = _lib.load()

    def quantize(w=ONE, dtype=BF16, E=2, K=64, N=8, se=512, ldw=64, group=32, packed=ONE, scales=ONE):
        return lib.ela_expert_quantize(w, dtype, E, K, N, se, ldw, group, packed, scales, NULL)

    for bad in (dict(dtype=F32), dict(E=0), dict(E=4097), dict(K=0), dict(N=0), dict(group=16), dict(group=100), dict(se=-1), dict(ldw=-1), dict(w=NULL),
                dict(packed=NULL), dict(scales=NULL), dict(w=ODD), dict(scales=ODD), dict(packed=ctypes.c_void_p(264))):
        assert quantize(**bad) == ARGUMENT, bad
    assert quantize(E=4096, N=1 << 30, K=1 << 30) == _lib.ELA_ERR_UNSUPPORTED

    def dequantize(packed=ONE, scales=ONE, dtype=BF16, E=2, K=64, N=8, group=32, w=ONE):
        return lib.ela_expert_dequantize(packed, scales, dtype, E, K, N, group, w, NULL)

    for bad in (dict(dtype=F32), dict(E=0), dict(K=0), dict(N=0), dict(group=0), dict(w=NULL), dict(packed=NULL), dict(scales=NULL), dict(w=ODD),
                dict(scales=ODD), dict(packed=ctypes.c_void_p(260))):
        assert dequantize(**bad) == ARGUMENT, bad

    def linear(x=ONE, packed=ONE, scales=ONE, bias=NULL, res=NULL, off=ONE, dtype=BF16, R=4, E=2, K=64, N=8, group=32, ldx=64, ldr=8, act=0, y=ONE):
        return lib.ela_expert_linear_4bit(x, packed, scales, bias, res, off, dtype, R, E, K, N, group, ldx, ldr, act, y, NULL, 0, NULL)

    for bad in (dict(dtype=F32), dict(R=-1), dict(E=0), dict(E=4097), dict(K=0), dict(N=0), dict(group=31), dict(ldx=-1), dict(ldr=-1), dict(act=4),
                dict(act=-1), dict(x=NULL), dict(packed=NULL), dict(scales=NULL), dict(y=NULL), dict(off=NULL), dict(x=ODD), dict(scales=ODD), dict(bias=ODD),
                dict(res=ODD), dict(y=ODD), dict(off=HALF), dict(packed=ctypes.c_void_p(272 - 8))):
        assert linear(**bad) == ARGUMENT, bad
    assert linear(R=0, x=NULL) == _lib.ELA_OK


def test_shapes_that_a_traced_graph_sees():
    with FakeTensorMode():
        l = torch.empty(5, 12, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        expert, weights = ela.expert_route(l, 3)
        assert expert.shape == weights.shape == (5, 3) and expert.dtype == torch.int32 and weights.dtype == torch.float32
        assert weights.requires_grad and not expert.requires_grad
        d = torch.ops.ela_native.expert_route_grad(torch.empty(5, 3, device="cuda"), l.detach(), expert, 0, True, 1.0)
        assert d.shape == l.shape and d.dtype == l.dtype
        w = torch.empty(2, 10, 100, dtype=torch.float16, device="cuda")
        q = ela.expert_quantize(w, 32)
        assert q.packed.shape == (2, 10, 16) and q.scales.shape == (2, 4, 10) and ela.expert_dequantize(q).shape == w.shape
        one = ela.expert_quantize(w[0], 32)
        assert one.packed.shape == (10, 16) and ela.expert_dequantize(one).shape == (10, 100)
        y = ela.expert_linear_4bit(torch.empty(7, 100, dtype=torch.float16, device="cuda"), one)
        assert y.shape == (7, 10) and y.dtype == torch.float16


def test_gradients_that_would_be_lost_are_refused():
    import torch.autograd.forward_ad as fwd
    with FakeTensorMode():
        w = torch.empty(2, 16, 64, dtype=torch.bfloat16, device="cuda")
        q = ela.expert_quantize(w, 32)
        x, off = torch.empty(4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
        l = torch.empty(4, 8, device="cuda")
        calls = [(lambda v: ela.expert_quantize(v, 32), w), (lambda v: ela.expert_dequantize(q._replace(scales=v)), q.scales),
                 (lambda v: ela.expert_linear_4bit(v, q, offsets=off), x),
                 (lambda v: ela.expert_linear_4bit(x, q._replace(scales=v), offsets=off), q.scales)]
        for f, v in calls:
            f(v)
            leaf = torch.empty_like(v).requires_grad_()
            with pytest.raises(RuntimeError, match="no gradient"):
                f(leaf)
            with torch.no_grad():
                f(leaf)
        for f, v in calls + [(lambda v: ela.expert_route(v, 2), l)]:
            with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                f(fwd.make_dual(v, torch.empty_like(v)))
