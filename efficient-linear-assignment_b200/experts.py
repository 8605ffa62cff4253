"""The expert layer around an assignment of tokens to experts.

``linear_assignment`` (or any router) says which expert each token goes to;
these operators take the tokens there and back:

    plan = expert_plan(expert, num_experts)          # stable sort by expert
    rows = expert_dispatch(x, plan)                  # tokens in expert order
    h    = expert_linear(rows, w1, b1, activation="gelu", offsets=plan.offsets)
    h    = expert_linear(h, w2, b2, offsets=plan.offsets)
    out  = expert_combine(h, plan, weights)          # back, weighted and summed

All of them are C++ torch operators (csrc/ela_expert_op.cpp) over the C ABI of
include/ela_expert.h, which also checks the arguments (TypeError, ValueError,
RuntimeError for host tensors): current stream, no synchronisation, no data-dependent
sizes, so the whole layer can be captured in a CUDA graph.  Dispatch, combine
and linear are differentiable (once, in reverse mode).  A choice outside [0, num_experts), such
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
MAX_EXPERTS = 4096  # ELA_EXPERT_MAX


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
    """The operators' overloads (loaded once: the lookup by name costs host time)."""
    global _ops
    if _ops is None:
        _native_op()  # loads the operator library
        n = torch.ops.ela_native
        _ops = (n.expert_plan.default, n.expert_dispatch.default, n.expert_combine.default, n.expert_linear.default)
    return _ops


def expert_plan(expert: torch.Tensor, num_experts: int) -> ExpertPlan:
    """Stable sort of the choices ``expert`` (T,) or (T, k), int32 or int64, by
    expert.  Choices outside [0, num_experts) go last."""
    return ExpertPlan._make((_ops or _native())[0](expert, num_experts))


def expert_dispatch(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """Token rows ``x`` (T, H) in expert order, (T*k, H): row r is the token of
    slot ``plan.source[r]``; rows of no expert are zeros.  fp32, fp16 or bf16.
    Backward: each token's gradients summed in fp32, rounded once."""
    return (_ops or _native())[1](x, plan[1], plan[0])


def expert_combine(y: torch.Tensor, plan: ExpertPlan, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows ``y`` (T*k, H) back to their tokens, (T, H): the sum over a token's
    choices of weight times row, in fp32, rounded once.  weights (T, k) (or (T,)
    when k is 1), float32 or y's dtype; None: 1.  Choices of no expert add
    nothing.  Backward: gradients of y and of weights."""
    return (_ops or _native())[2](y, plan[1], plan[0], weights)


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
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"expert_linear: unknown activation '{activation}'. Options: {list(ACTIVATIONS)}")
    return (_ops or _native())[3](x, weight, bias, residual, offsets, code)


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
                weights.new_empty(weights.shape) if need_w else dout.new_empty((0,)))

    @torch.library.register_fake("ela_native::expert_linear_z")
    def _(x, weight, bias, residual, offsets, activation, want_z):
        kept = torch.float32 if activation in (ACTIVATIONS["gelu"], ACTIVATIONS["silu"]) else x.dtype
        return x.new_empty((x.shape[0], weight.shape[-2])), x.new_empty((x.shape[0] if want_z else 0, weight.shape[-2]), dtype=kept)

    @torch.library.register_fake("ela_native::expert_linear_grad")
    def _(dy, z, x, weight, offsets, activation, wsizes, bsizes, need_x, need_w, need_b):
        return (dy.new_empty((dy.shape[0] if need_x else 0, wsizes[-1])), dy.new_empty(wsizes if need_w else (0,)),
                dy.new_empty(bsizes if need_b else (0,)))


_register_fakes()
