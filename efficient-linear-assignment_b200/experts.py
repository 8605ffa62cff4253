"""The expert layer around an assignment of tokens to experts.

``linear_assignment`` (or any router) says which expert each token goes to;
these operators take the tokens there and back:

    plan = expert_plan(expert, num_experts)          # stable sort by expert
    rows = expert_dispatch(x, plan)                  # tokens in expert order
    h    = expert_linear(rows, w1, b1, activation="gelu", offsets=plan.offsets)
    h    = expert_linear(h, w2, b2, offsets=plan.offsets)
    out  = expert_combine(h, plan, weights)          # back, weighted and summed

All of them are C++ torch operators (csrc/ela_expert_op.cpp) over the C ABI of
include/ela_expert.h: current stream, no synchronisation, no data-dependent
sizes, so the whole layer can be captured in a CUDA graph.  Dispatch, combine
and linear are differentiable (once).  A choice outside [0, num_experts), such
as the solver's -1 for an unassigned row, belongs to no expert: it takes one of
the last rows, is dispatched as zeros and adds nothing to the combined token.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .solver import _native_op

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
MAX_EXPERTS = 4096

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


class ExpertPlan(NamedTuple):
    """Where the slots (token t, choice j) go.

    offsets   int32 (E+1,): expert e has rows offsets[e] .. offsets[e+1]
    position  int32 (T, k): the row of each slot; offsets[E] and later: no expert
    source    int32 (T*k,): the slot t*k + j of each row
    """
    offsets: torch.Tensor
    position: torch.Tensor
    source: torch.Tensor


_ops = None


def _native():
    global _ops
    if _ops is None:
        _native_op()  # loads the operator library
        _ops = torch.ops.ela_native
    return _ops


def _need_cuda(name: str, t: torch.Tensor) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{name} needs CUDA tensors (there is no CPU path)")


def expert_plan(expert: torch.Tensor, num_experts: int) -> ExpertPlan:
    """Stable sort of the choices ``expert`` (T,) or (T, k), int32 or int64, by
    expert.  Choices outside [0, num_experts) go last."""
    _need_cuda("expert_plan", expert)
    if expert.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"expert must be int32 or int64, not {expert.dtype}")
    if expert.dim() not in (1, 2):
        raise ValueError("expert must be (T,) or (T, k)")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be 1..{MAX_EXPERTS}")
    if expert.numel() >= 1 << 31:
        raise ValueError("more than 2^31 - 1 choices")
    return ExpertPlan(*_native().expert_plan(expert, num_experts))


def _check_plan(name: str, plan: ExpertPlan, t: torch.Tensor) -> None:
    _need_cuda(name, t)
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name}: unsupported dtype {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name}: rows must be a matrix")
    if plan.position.dim() != 2 or plan.position.dtype != torch.int32 or plan.offsets.dtype != torch.int32:
        raise ValueError(f"{name}: plan.position must be int32 (T, k), plan.offsets int32 (E+1,)")


def expert_dispatch(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """Token rows ``x`` (T, H) in expert order, (T*k, H): row r is the token of
    slot ``plan.source[r]``; rows of no expert are zeros.  fp32, fp16 or bf16.
    Backward: each token's gradients summed in fp32, rounded once."""
    _check_plan("expert_dispatch", plan, x)
    if x.shape[0] != plan.position.shape[0]:
        raise ValueError(f"expert_dispatch: x has {x.shape[0]} tokens, the plan {plan.position.shape[0]}")
    return _native().expert_dispatch(x, plan.position, plan.offsets)


def expert_combine(y: torch.Tensor, plan: ExpertPlan, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows ``y`` (T*k, H) back to their tokens, (T, H): the sum over a token's
    choices of weight times row, in fp32, rounded once.  weights (T, k) (or (T,)
    when k is 1), float32 or y's dtype; None: 1.  Choices of no expert add
    nothing.  Backward: gradients of y and of weights."""
    _check_plan("expert_combine", plan, y)
    if y.shape[0] != plan.position.numel():
        raise ValueError(f"expert_combine: y has {y.shape[0]} rows, the plan {plan.position.numel()}")
    if weights is not None:
        if weights.dtype != torch.float32 and weights.dtype != y.dtype:
            raise TypeError(f"expert_combine: weights must be float32 or {y.dtype}, not {weights.dtype}")
        if weights.dim() == 1 and plan.position.shape[1] == 1:
            weights = weights.unsqueeze(1)
        if weights.shape != plan.position.shape or weights.device != y.device:
            raise ValueError("expert_combine: weights must be (T, k) on y's device")
    return _native().expert_combine(y, plan.position, plan.offsets, weights)


def expert_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None, activation: str = "none",
                  offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x W_e^T + b_e) + residual`` for the rows of each expert, (R, N).

    x (R, K); weight (E, N, K), or (N, K) for one matrix; bias (E, N) or (N,);
    residual (R, N); activation "none", "relu", "gelu" (erf) or "silu"; offsets
    int32 (E+1,): expert e has rows offsets[e] .. offsets[e+1] (None: every row
    is the one expert's).  Rows of no expert get the residual, or 0.  fp16 or
    bf16; sums in fp32 on the tensor cores, one rounding at the end.  Backward:
    gradients of x, weight, bias and residual."""
    _need_cuda("expert_linear", x)
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"expert_linear: x must be float16 or bfloat16, not {x.dtype}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"expert_linear: unknown activation '{activation}'. Options: {list(ACTIVATIONS)}")
    if x.dim() != 2 or weight.dim() not in (2, 3) or weight.shape[-1] != x.shape[1]:
        raise ValueError("expert_linear: x must be (R, K), weight (E, N, K) or (N, K)")
    E, N = (weight.shape[0] if weight.dim() == 3 else 1), weight.shape[-2]
    if min(E, N, x.shape[1]) < 1 or E > MAX_EXPERTS:
        raise ValueError(f"expert_linear: E must be 1..{MAX_EXPERTS}, N and K at least 1")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"expert_linear: {name} must be {x.dtype}, not {t.dtype}")
        if t is not None and t.device != x.device:
            raise ValueError(f"expert_linear: {name} must be on x's device")
    if bias is not None and tuple(bias.shape) != ((E, N) if weight.dim() == 3 else (N,)):
        raise ValueError("expert_linear: bias must be (E, N), or (N,) for one matrix")
    if residual is not None and tuple(residual.shape) != (x.shape[0], N):
        raise ValueError("expert_linear: residual must be (R, N)")
    if offsets is None:
        if E != 1:
            raise ValueError("expert_linear: offsets are needed for more than one expert")
    elif offsets.dtype != torch.int32 or tuple(offsets.shape) != (E + 1,) or offsets.device != x.device:
        raise ValueError("expert_linear: offsets must be int32 (E+1,) on x's device")
    return _native().expert_linear(x, weight, bias, residual, offsets, ACTIVATIONS[activation])


def expert_check() -> None:
    """Raise AuctionError if a product on the current device gave up a wait since
    the last check (its results are then incomplete).  Waits for the device; the
    operators themselves never do."""
    status = ctypes.c_int(0)
    _lib.check(_lib.load().ela_expert_status(ctypes.byref(status)), "ela_expert_status")
    _lib.check(status.value, "expert_linear kernel")


def _register_fakes() -> None:
    try:
        _native()
    except ImportError:
        return

    @torch.library.register_fake("ela_native::expert_plan")
    def _(expert, num_experts):
        shape = expert.shape if expert.dim() == 2 else (expert.shape[0], 1)
        new = lambda s: expert.new_empty(s, dtype=torch.int32)  # noqa: E731
        return new((num_experts + 1,)), new(shape), new((expert.numel(),))

    @torch.library.register_fake("ela_native::expert_dispatch")
    def _(x, position, offsets):
        return x.new_empty((position.numel(), x.shape[1]))

    @torch.library.register_fake("ela_native::expert_combine")
    def _(y, position, offsets, weights):
        return y.new_empty((position.shape[0], y.shape[1]))

    @torch.library.register_fake("ela_native::expert_linear")
    def _(x, weight, bias, residual, offsets, activation):
        return x.new_empty((x.shape[0], weight.shape[-2]))

    @torch.library.register_fake("ela_native::expert_combine_grad")
    def _(dout, y, position, offsets, weights, need_y, need_w):
        return (dout.new_empty((position.numel() if need_y else 0, dout.shape[1])),
                weights.new_empty(position.shape) if need_w else dout.new_empty((0,)))

    @torch.library.register_fake("ela_native::expert_linear_z")
    def _(x, weight, bias, residual, offsets, activation, want_z):
        return x.new_empty((x.shape[0], weight.shape[-2])), x.new_empty((x.shape[0] if want_z else 0, weight.shape[-2]))

    @torch.library.register_fake("ela_native::expert_linear_grad")
    def _(dy, z, x, weight, offsets, activation, wsizes, bsizes, need_x, need_w, need_b):
        return (dy.new_empty((dy.shape[0] if need_x else 0, wsizes[-1])), dy.new_empty(wsizes if need_w else (0,)),
                dy.new_empty(bsizes if need_b else (0,)))


_register_fakes()
