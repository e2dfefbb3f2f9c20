"""Rows sorted by expert and back, with weights applied, and a block of fused
MLP experts (no counterpart in the reference, which has one MLP).

* ``expert_sort(ids, num_experts)`` -- the plan of a batch: where each slot
  (token, choice) lies when the slots are ordered by expert;
* ``expert_dispatch(x, plan)`` -- each token's row copied to its slots' rows;
* ``expert_combine(y, weights, plan)`` -- the weighted sum of its slots' rows
  back at each token;
* ``FusedMLPExperts`` -- norm, router, dispatch, a FusedMLPSoftplus for each
  expert, combine.

Rows are fp16, bf16 or fp32 of any width; sums are fp32 in a fixed order, so
results are the same from run to run.  Everything runs on the current CUDA
stream; the three calls never make the host wait, FusedMLPExperts does once a
call.  There is no CPU path.  Eager calls go through
the native binding (_native.py); under torch.compile, tracers and dispatch modes
and on fake tensors the calls are the operators ``torch.ops.mlpk.expert_*``.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib
from ._native import native
from .modules import FusedMLPSoftplus
from .norm import DTYPES, FusedRMSNorm, _eager, _needs_grad, _refuse_transforms


class ExpertPlan(NamedTuple):
    """Where the slots of a batch lie in the order by expert (int32, on the
    GPU).  ``row_of[t, k]`` is the row of token t's k-th choice;
    ``offsets[e]`` is expert e's first row and ``offsets[-1]`` the number of
    rows kept.  Slots without an expert lie behind those."""

    row_of: Tensor
    offsets: Tensor

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def counts(self) -> Tensor:
        """Rows of each expert."""
        return self.offsets.diff()


# ------------------------------------------------------------ torch.ops.mlpk
def _require_cuda(*ts):
    for t in ts:
        if isinstance(t, Tensor) and not t.is_cuda:
            raise RuntimeError("the expert operators run on CUDA (sm_100) only; got a CPU tensor")


def _check_ids(ids, num_experts) -> None:
    if not isinstance(ids, Tensor) or ids.dim() != 2:
        raise ValueError("ids must be a 2-D tensor [tokens, choices]")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if not 1 <= num_experts <= _lib.EXPERT_MAX:
        raise ValueError(f"num_experts must be 1 to {_lib.EXPERT_MAX}, got {num_experts}")
    if ids.shape[1] < 1 or ids.numel() > 2 ** 31 - 1:
        raise ValueError(f"ids must have at least one choice a token and at most 2^31 - 1 slots, got {tuple(ids.shape)}")


def _check_rows(what: str, t, of_slots: bool, row_of, offsets) -> None:
    """A tensor with a row for each slot, or each token, of a plan."""
    if row_of.dim() != 2 or row_of.dtype != torch.int32 or row_of.shape[1] < 1 or offsets.dim() != 1 or \
            offsets.dtype != torch.int32 or offsets.shape[0] < 2 or not offsets.is_contiguous():
        raise ValueError("plan must be what expert_sort returned")
    rows = row_of.numel() if of_slots else row_of.shape[0]
    if not isinstance(t, Tensor) or t.dim() != 2 or t.shape[0] != rows or t.shape[1] < 1:
        raise ValueError(f"{what} must be a 2-D tensor of {rows} rows")
    if t.dtype not in DTYPES:
        raise TypeError(f"{what} must be fp16, bf16 or fp32, got {t.dtype}")
    if t.device != row_of.device or t.device != offsets.device:
        raise ValueError(f"{what} is on {t.device}, the plan on {row_of.device} and {offsets.device}")


def _check_combine(y, weights, row_of, offsets) -> None:
    _check_rows("y", y, True, row_of, offsets)
    if weights is not None and (weights.shape != row_of.shape or weights.device != y.device
                                or (weights.dtype != y.dtype and weights.dtype != torch.float32)):
        raise ValueError(f"weights must be a {tuple(row_of.shape)} tensor of {y.dtype} or float32 on {y.device}")


def _check_combine_bwd(grad_out, y, weights, row_of, offsets, want_dw) -> None:
    _check_combine(y, weights, row_of, offsets)
    if grad_out.shape != (row_of.shape[0], y.shape[1]) or grad_out.dtype != y.dtype or grad_out.device != y.device:
        raise ValueError(f"grad_out must be a {(row_of.shape[0], y.shape[1])} {y.dtype} tensor on {y.device}")
    if want_dw and weights is None:
        raise ValueError("there are no weights to have a gradient")


@torch.library.custom_op("mlpk::expert_sort", mutates_args=())
def _sort_op(ids: Tensor, num_experts: int) -> list[Tensor]:
    _require_cuda(ids)
    _check_ids(ids, num_experts)
    return list(native().sort_ids(ids, num_experts))


@_sort_op.register_fake
def _sort_fake(ids, num_experts):
    _check_ids(ids, num_experts)
    return [ids.new_empty(ids.shape, dtype=torch.int32), ids.new_empty((num_experts + 1,), dtype=torch.int32)]


@torch.library.custom_op("mlpk::expert_dispatch", mutates_args=())
def _dispatch_op(x: Tensor, row_of: Tensor, offsets: Tensor) -> Tensor:
    _require_cuda(x, row_of, offsets)
    _check_rows("x", x, False, row_of, offsets)
    return native().dispatch_rows(x, row_of, offsets)


@_dispatch_op.register_fake
def _dispatch_fake(x, row_of, offsets):
    _check_rows("x", x, False, row_of, offsets)
    return x.new_empty((row_of.shape[0] * row_of.shape[1], x.shape[1]))


@torch.library.custom_op("mlpk::expert_combine", mutates_args=())
def _combine_op(y: Tensor, weights: Optional[Tensor], row_of: Tensor, offsets: Tensor) -> Tensor:
    _require_cuda(y, weights, row_of, offsets)
    _check_combine(y, weights, row_of, offsets)
    return native().combine_rows(y, weights, row_of, offsets)


@_combine_op.register_fake
def _combine_fake(y, weights, row_of, offsets):
    _check_combine(y, weights, row_of, offsets)
    return y.new_empty((row_of.shape[0], y.shape[1]))


@torch.library.custom_op("mlpk::expert_combine_bwd", mutates_args=())
def _combine_bwd_op(grad_out: Tensor, y: Tensor, weights: Optional[Tensor], row_of: Tensor, offsets: Tensor,
                    want_dy: bool, want_dw: bool) -> list[Tensor]:
    """[dy] and / or [dw], as wanted."""
    _require_cuda(grad_out, y, weights, row_of, offsets)
    _check_combine_bwd(grad_out, y, weights, row_of, offsets, want_dw)
    dy, dw = native().combine_backward(grad_out, y, weights, row_of, offsets, want_dy, want_dw)
    return ([dy] if want_dy else []) + ([dw] if want_dw else [])


@_combine_bwd_op.register_fake
def _combine_bwd_fake(grad_out, y, weights, row_of, offsets, want_dy, want_dw):
    _check_combine_bwd(grad_out, y, weights, row_of, offsets, want_dw)
    return ([y.new_empty(y.shape)] if want_dy else []) + ([weights.new_empty(weights.shape)] if want_dw else [])


# ------------------------------------------------------------ autograd
class _DispatchFn(torch.autograd.Function):
    """The node that tracers and modes see (as _CombineFn).  Its gradient is an
    operator without a derivative: asking for one raises."""

    @staticmethod
    def forward(ctx, x, row_of, offsets):
        ctx.save_for_backward(row_of, offsets)
        return torch.ops.mlpk.expert_dispatch(x, row_of, offsets)

    @staticmethod
    def backward(ctx, grad):
        _refuse_transforms("the gradient of expert_dispatch", grad)
        return torch.ops.mlpk.expert_combine(grad, None, *ctx.saved_tensors), None, None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, row_of, offsets):
        ctx.save_for_backward(y, weights, row_of, offsets)
        return torch.ops.mlpk.expert_combine(y, weights, row_of, offsets)

    @staticmethod
    def backward(ctx, grad):
        y, weights, row_of, offsets = ctx.saved_tensors
        _refuse_transforms("the gradient of expert_combine", grad, y, weights)
        want_dy, want_dw = ctx.needs_input_grad[0], weights is not None and ctx.needs_input_grad[1]
        if not want_dw:  # dy does not depend on y, nor dw on the weights
            y = y.detach()
        if not want_dy:
            weights = weights.detach()
        got = torch.ops.mlpk.expert_combine_bwd(grad, y, weights, row_of, offsets, want_dy, want_dw)
        return got[0] if want_dy else None, got[-1] if want_dw else None, None, None


# ------------------------------------------------------------ public calls
def expert_sort(ids: Tensor, num_experts: int) -> ExpertPlan:
    """The plan of a batch from the experts its tokens chose.

    ``ids`` is an int32 or int64 CUDA tensor ``[tokens, choices]``; the order is
    stable (by expert, then by token and choice).  A slot whose id is outside
    ``[0, num_experts)`` -- -1 for a choice over its expert's capacity, say -- is
    dropped: dispatch gives it a row of zeros behind the kept rows, combine
    leaves it out.  At most 1024 experts and 2^31 - 1 slots.
    """
    if _eager(ids):
        got = native().expert_sort(ids, num_experts)
        if got is not None:
            return ExpertPlan(*got)
    _refuse_transforms("expert_sort", ids)
    _require_cuda(ids)
    _check_ids(ids, num_experts)
    return ExpertPlan(*torch.ops.mlpk.expert_sort(ids, num_experts))


def expert_dispatch(x: Tensor, plan: ExpertPlan) -> Tensor:
    """``[tokens * choices, width]``: row ``plan.row_of[t, k]`` is ``x[t]``, rows
    of dropped slots are zero.  Differentiable in x (a sum over the kept slots)."""
    if _eager(x):
        got = native().expert_dispatch(x, *plan)
        if got is not None:
            return got
    _refuse_transforms("expert_dispatch", x, *plan)
    _require_cuda(x, *plan)
    _check_rows("x", x, False, *plan)
    if _needs_grad(x):
        return _DispatchFn.apply(x, *plan)
    return torch.ops.mlpk.expert_dispatch(x, *plan)


def expert_combine(y: Tensor, weights: Optional[Tensor], plan: ExpertPlan) -> Tensor:
    """``[tokens, width]``: the sum over k of ``weights[t, k] * y[plan.row_of[t, k]]``
    in fp32; dropped slots add nothing, whatever their rows and weights hold.
    ``weights`` is ``[tokens, choices]`` in y's dtype or fp32, or None for ones.
    Differentiable in y and weights."""
    if _eager(y):
        got = native().expert_combine(y, weights, *plan)
        if got is not None:
            return got
    _refuse_transforms("expert_combine", y, weights, *plan)
    _require_cuda(y, weights, *plan)
    _check_combine(y, weights, *plan)
    if _needs_grad(y, weights):
        return _CombineFn.apply(y, weights, *plan)
    return torch.ops.mlpk.expert_combine(y, weights, *plan)


class FusedMLPExperts(nn.Module):
    """A residual block of fused MLP experts: ``h = x + residual``, an RMS norm of
    h, a router that takes each row's ``top`` best experts, a FusedMLPSoftplus
    ``D -> H -> .. -> D`` for each expert, and the weighted sum of their rows.

    ``forward(x, residual=None)`` returns ``(out, h)``, the next block's x and
    residual.  ``capacity`` (rows an expert takes, the first of a batch; None:
    all) drops the choices above it.  Each expert runs on its own rows: their
    numbers are read by the host, once a call.
    """

    def __init__(self, D: int = 128, H: int = 128, num_experts: int = 8, top: int = 2, num_layers: int = 3,
                 capacity: Optional[int] = None, eps: float = 1e-6):
        super().__init__()
        if not 1 <= top <= num_experts:
            raise ValueError(f"top must be 1 to num_experts, got {top}")
        if capacity is not None and capacity < 1:
            raise ValueError(f"capacity must be positive, got {capacity}")
        self.top, self.capacity = top, capacity
        self.norm = FusedRMSNorm(D, eps)
        self.router = nn.Parameter(torch.empty(D, num_experts).uniform_(-1 / math.sqrt(D), 1 / math.sqrt(D)))
        self.experts = nn.ModuleList(FusedMLPSoftplus(D=D, H=H, out_features=D, num_layers=num_layers)
                                     for _ in range(num_experts))

    def forward(self, x: Tensor, residual: Optional[Tensor] = None):
        y, h = self.norm(x, residual) if residual is not None else (self.norm(x), x)
        scores, ids = (y.float() @ self.router.float()).topk(self.top, dim=1)
        weights = torch.softmax(scores, dim=1)
        plan = expert_sort(ids, len(self.experts))
        if self.capacity is not None:
            rank = plan.row_of - plan.offsets[:-1][ids]
            plan = expert_sort(torch.where(rank < self.capacity, ids, -1), len(self.experts))
        rows = expert_dispatch(y, plan)
        counts = plan.counts.tolist()
        *parts, dropped = rows.split([*counts, rows.shape[0] - sum(counts)])
        parts = [expert(part).to(rows.dtype) if len(part) else part for expert, part in zip(self.experts, parts)]
        return expert_combine(torch.cat([*parts, dropped]), weights, plan), h
