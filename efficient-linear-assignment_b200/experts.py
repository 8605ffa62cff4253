"""The expert layer around an assignment of tokens to experts.

``linear_assignment`` (or any router) says which expert each token goes to;
these operators take the tokens there and back:

    plan = expert_plan(expert, num_experts)          # stable sort by expert
    rows = expert_dispatch(x, plan)                  # tokens in expert order
    h    = expert_linear(rows, w1, b1, activation="gelu", offsets=plan.offsets)
    h    = expert_linear(h, w2, b2, offsets=plan.offsets)
    out  = expert_combine(h, plan, weights)          # back, weighted and summed

Beside the solver, ``expert_route`` makes the choices and their weights from a router's
logits; for serving, ``expert_quantize`` brings the experts to 4 bits and
``expert_linear_4bit`` multiplies with them:

    expert, weights = expert_route(logits, 2)
    w1 = expert_quantize(w1, group=64)               # once
    h  = expert_linear_4bit(rows, w1, b1, activation="gelu", offsets=plan.offsets)

All of them are C++ torch operators (csrc/ela_expert_op.cpp) over the C ABI of
include/ela_expert.h, which also checks the arguments (TypeError, ValueError,
RuntimeError for host tensors): current stream, no synchronisation, no data-dependent
sizes, so the whole layer can be captured in a CUDA graph.  Route, dispatch, combine
and linear are differentiable (once, in reverse mode); the 4-bit operators serve, and raise
where a gradient would be lost.  A choice outside [0, num_experts), such
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
SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "top2": 1}
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


class ExpertRoute(NamedTuple):
    """The experts of each token and their weights.

    expert   int32 (T, k): the best first; -1 where none is left
    weights  float32 (T, k): 0 where the expert is -1
    """
    expert: torch.Tensor
    weights: torch.Tensor


class Expert4Bit(NamedTuple):
    """Experts' weights (E, N, K), or one matrix (N, K), in 4 bits: weight k of a row is
    q * scale, q in -8..7, rounded to the scale's type; ``group`` inputs share a scale.

    packed    int32 (E, N, W), W = 8 * ceil(K / 64): word i of a row holds q + 8 of the inputs
              8 i + j at bits 4 * (j // 2) + 16 * (j % 2); inputs from K on are q = 0
    scales    (E, ceil(K / group), N), float16 or bfloat16
    features  K
    group     32, 64 or 128
    """
    packed: torch.Tensor
    scales: torch.Tensor
    features: int
    group: int


_ops = None


def _native():
    """The operators' overloads (loaded once: the lookup by name costs host time)."""
    global _ops
    if _ops is None:
        _native_op()  # loads the operator library
        n = torch.ops.ela_native
        _ops = (n.expert_plan.default, n.expert_dispatch.default, n.expert_combine.default, n.expert_linear.default,
                n.expert_route.default, n.expert_quantize.default, n.expert_dequantize.default,
                n.expert_linear_4bit.default)
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


def expert_route(logits: torch.Tensor, k: int, score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
                 groups_kept: Optional[int] = None, group_score: str = "max", renormalize: bool = True,
                 scale: float = 1.0) -> ExpertRoute:
    """The ``k`` best experts of each token and their weights, from ``logits`` (T, E).

    Scores are the row's softmax or sigmoid.  Experts are chosen by score, or by
    score + ``bias`` (float32 (E,), which balances the choice and does not touch the
    weights); with ``groups`` > 1 only among the experts of the ``groups_kept`` best of
    the equal runs of experts, ranked by their best expert ("max") or the sum of their two
    best ("top2").  The weights are the chosen scores, divided by their sum with
    ``renormalize``, times ``scale``.  Ties go to the lowest index, NaN counts as the
    largest, and the order is that of 64-bit arithmetic.  An expert whose logit (or bias)
    is -inf is never chosen: a token without enough others in the groups that stay gets expert -1,
    weight 0.  By "top2" a group with one open expert ranks with the closed ones, after every
    group with two, so that its expert may be left out.
    fp32, fp16 or bf16; k up to 64.  Backward: the gradient of the logits."""
    code, by = SCORES.get(score), GROUP_SCORES.get(group_score)
    if code is None:
        raise ValueError(f"expert_route: unknown score '{score}'. Options: {list(SCORES)}")
    if by is None:
        raise ValueError(f"expert_route: unknown group_score '{group_score}'. Options: {list(GROUP_SCORES)}")
    return ExpertRoute._make((_ops or _native())[4](logits, k, code, bias, groups, groups if groups_kept is None else groups_kept,
                                                    by, renormalize, scale))


def expert_quantize(weight: torch.Tensor, group: int = 64) -> Expert4Bit:
    """``weight`` (E, N, K) or (N, K), fp16 or bf16, in 4 bits with a scale for every
    ``group`` (32, 64 or 128) inputs of a row: scale = max|w| / 7, rounded to the weight's
    type, q = w / scale rounded to even.  A group with a NaN or an infinity gets a scale
    that is one.  No gradient."""
    return Expert4Bit(*(_ops or _native())[5](weight, group), weight.shape[-1], group)


def expert_dequantize(weight: Expert4Bit) -> torch.Tensor:
    """The weights that ``weight`` stands for, (E, N, K) or (N, K), in the scales' type."""
    return (_ops or _native())[6](*weight)


def expert_linear_4bit(x: torch.Tensor, weight: Expert4Bit, bias: Optional[torch.Tensor] = None,
                       residual: Optional[torch.Tensor] = None, activation: str = "none",
                       offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``expert_linear`` with 4-bit weights: ``act(x W_e^T + b_e) + residual`` where W is what
    ``expert_dequantize(weight)`` returns, without writing it.  x, bias and residual in the
    scales' type; the other arguments, the rows of no expert and the sums in fp32 are as there.
    No gradient: raises where one is asked for."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"expert_linear_4bit: unknown activation '{activation}'. Options: {list(ACTIVATIONS)}")
    return (_ops or _native())[7](x, *weight, bias, residual, offsets, code)


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


    @torch.library.register_fake("ela_native::expert_route")
    def _(logits, k, score, bias, groups, groups_kept, group_score, renormalize, scale):
        shape = (logits.shape[0], k)
        return logits.new_empty(shape, dtype=torch.int32), logits.new_empty(shape, dtype=torch.float32)

    @torch.library.register_fake("ela_native::expert_route_grad")
    def _(dweights, logits, expert, score, renormalize, scale):
        return logits.new_empty(logits.shape)

    @torch.library.register_fake("ela_native::expert_quantize")
    def _(weight, group):
        *lead, n, k = weight.shape
        return (weight.new_empty((*lead, n, (k + 63) // 64 * 8), dtype=torch.int32),
                weight.new_empty((*lead, (k + group - 1) // group, n)))

    @torch.library.register_fake("ela_native::expert_dequantize")
    def _(packed, scales, features, group):
        return scales.new_empty((*packed.shape[:-1], features))

    @torch.library.register_fake("ela_native::expert_linear_4bit")
    def _(x, packed, scales, features, group, bias, residual, offsets, activation):
        return x.new_empty((x.shape[0], packed.shape[-2]))


_register_fakes()
