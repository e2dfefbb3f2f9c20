"""Root-mean-square norm with the residual's addition (no counterpart in the
reference, whose MLP takes its rows as they come).

* ``fused_rms_norm(x, weight, residual=r)`` -- ``h = x + r`` and
  ``y = h / sqrt(mean(h^2) + eps) * weight`` in one pass, differentiable;
* ``fused_rms_norm_fp8(...)`` -- the same with an 8-bit (e4m3) output and its
  fp32 scales, for inference;
* ``FusedRMSNorm`` -- the module.

x is fp16, bf16 or fp32 of shape ``[..., width]`` with width up to 32768; all
arithmetic is fp32.  The kernels run on the current CUDA stream; there is no
CPU path.  Eager calls go through the native binding (_native.py), whose
autograd nodes are native too; under torch.compile, tracers and dispatch modes and
on fake tensors the calls are the operators ``torch.ops.mlpk.rms_norm`` /
``rms_norm_bwd`` / ``rms_norm_fp8``.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn as nn
from torch import Tensor

from . import _lib
from ._native import native

DTYPES = {torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16}


def _eager(x) -> bool:
    """Whether the native calls may take x.  (They in turn leave it to the
    operators where a dispatch mode, a tracer or a transform is to see them.)"""
    return (type(x) is Tensor or type(x) is nn.Parameter) and not torch.compiler.is_compiling()


def _refuse_transforms(name: str, *ts) -> None:
    """Raises where a tangent, or a transform of torch.func, would be lost."""
    if torch.compiler.is_compiling():
        return
    for t in ts:
        if not isinstance(t, Tensor):
            continue
        if torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise RuntimeError(f"{name} has no rule for torch.func's transforms (vmap, grad, jvp and the like)")
        if forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward-mode derivative")


def _check_args(x, weight, residual, eps):
    """Types and shapes; tensors of any device, the same for all."""
    if not isinstance(x, Tensor) or x.dim() < 1:
        raise ValueError("x must be a tensor [..., width]")
    if x.dtype not in DTYPES:
        raise TypeError(f"fused_rms_norm takes fp16, bf16 or fp32; got {x.dtype}")
    width = x.shape[-1]
    if not 1 <= width <= _lib.NORM_MAX_WIDTH:
        raise ValueError(f"the width must be 1 to {_lib.NORM_MAX_WIDTH}, got {width}")
    if weight is not None and (weight.shape != (width,) or weight.device != x.device
                               or (weight.dtype != x.dtype and weight.dtype != torch.float32)):
        raise ValueError(f"weight must be a [{width}] tensor of {x.dtype} or float32 on {x.device}")
    _check_like("residual", residual, x)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")


def _check_like(what, t, x):
    if t is not None and (t.shape != x.shape or t.dtype != x.dtype or t.device != x.device):
        raise ValueError(f"{what} must be a {tuple(x.shape)} {x.dtype} tensor on {x.device}")


def _check_cuda(x):
    if isinstance(x, Tensor) and not x.is_cuda:
        raise RuntimeError("fused_rms_norm runs on CUDA (sm_100) only; got a CPU tensor")


def _check(x, weight, residual, eps):
    _check_cuda(x)
    _check_args(x, weight, residual, eps)


def _check_bwd(x, residual, weight, rstd, grad_y, grad_h, want_dw):
    _check_args(x, weight, residual, 0.0)
    _check_like("grad_y", grad_y, x)
    _check_like("grad_h", grad_h, x)
    rows = x.numel() // x.shape[-1]
    if rstd.shape != (rows,) or rstd.dtype != torch.float32 or rstd.device != x.device or not rstd.is_contiguous():
        raise ValueError(f"rstd must be a contiguous [{rows}] float32 tensor on {x.device}")
    if want_dw and weight is None:
        raise ValueError("there is no weight to have a gradient")


def _check_group(group):
    if group not in (0, _lib.NORM_GROUP):
        raise ValueError(f"group must be 0 (the row) or {_lib.NORM_GROUP}, got {group}")


# ------------------------------------------------------------ torch.ops.mlpk
@torch.library.custom_op("mlpk::rms_norm", mutates_args=())
def rms_norm(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float) -> list[Tensor]:
    """[y, rstd], and h with a residual."""
    _check(x, weight, residual, eps)
    y, h, rstd = native().norm_forward(x, weight, residual, eps)
    return [y, rstd] if residual is None else [y, rstd, h]


@rms_norm.register_fake
def _rms_norm_fake(x, weight, residual, eps):
    _check_args(x, weight, residual, eps)
    rstd = x.new_empty((x.numel() // x.shape[-1],), dtype=torch.float32)
    return [x.new_empty(x.shape), rstd] + ([] if residual is None else [x.new_empty(x.shape)])


@torch.library.custom_op("mlpk::rms_norm_bwd", mutates_args=())
def rms_norm_bwd(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], rstd: Tensor, grad_y: Tensor,
                 grad_h: Optional[Tensor], want_dw: bool) -> list[Tensor]:
    """[dx], and dw if wanted."""
    _check_cuda(x)
    _check_bwd(x, residual, weight, rstd, grad_y, grad_h, want_dw)
    dx, dw = native().norm_backward(x, residual, weight, rstd, grad_y, grad_h, want_dw)
    return [dx, dw] if want_dw else [dx]


@rms_norm_bwd.register_fake
def _rms_norm_bwd_fake(x, residual, weight, rstd, grad_y, grad_h, want_dw):
    _check_bwd(x, residual, weight, rstd, grad_y, grad_h, want_dw)
    return [x.new_empty(x.shape)] + ([weight.new_empty(weight.shape)] if want_dw else [])


@torch.library.custom_op("mlpk::rms_norm_fp8", mutates_args=())
def rms_norm_fp8(x: Tensor, weight: Optional[Tensor], residual: Optional[Tensor], eps: float,
                 group: int) -> list[Tensor]:
    """[q, scale], and h with a residual."""
    _check(x, weight, residual, eps)
    _check_group(group)
    return list(native().norm_fp8(x, weight, residual, eps, group))


@rms_norm_fp8.register_fake
def _rms_norm_fp8_fake(x, weight, residual, eps, group):
    _check_args(x, weight, residual, eps)
    _check_group(group)
    groups = -(-x.shape[-1] // group) if group else 1
    return [x.new_empty(x.shape, dtype=torch.float8_e4m3fn),
            x.new_empty((*x.shape[:-1], groups), dtype=torch.float32)] + \
        ([] if residual is None else [x.new_empty(x.shape)])


# ------------------------------------------------------------ autograd
class _RMSNormFn(torch.autograd.Function):
    """The node that tracers and modes see.  Its gradients are operators without a
    derivative: asking for one raises."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, rstd, *h = torch.ops.mlpk.rms_norm(x, weight, residual, eps)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, residual, weight, rstd)
        return (y, h[0]) if h else y

    @staticmethod
    def backward(ctx, grad_y, grad_h=None):
        x, residual, weight, rstd = ctx.saved_tensors
        _refuse_transforms("the gradient of fused_rms_norm", grad_y, grad_h, x, residual, weight)
        want_dw = weight is not None and ctx.needs_input_grad[1]
        if grad_y is None:  # y was not used: the norm adds nothing
            dx, dw = grad_h, torch.zeros_like(weight) if want_dw and grad_h is not None else None
        else:
            if not (ctx.needs_input_grad[0] or ctx.needs_input_grad[2]):
                weight = weight.detach()  # dw alone, which does not depend on it
            dx, *dws = torch.ops.mlpk.rms_norm_bwd(x, residual, weight, rstd, grad_y, grad_h, want_dw)
            dw = dws[0] if dws else None
        return (dx if ctx.needs_input_grad[0] else None, dw,
                dx if residual is not None and ctx.needs_input_grad[2] else None, None)


def _needs_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def fused_rms_norm(x: Tensor, weight: Optional[Tensor] = None, *, residual: Optional[Tensor] = None,
                   eps: float = 1e-6):
    """``y = h * rsqrt(mean(h^2) + eps) * weight`` with ``h = x + residual``.

    Returns ``y``, or ``(y, h)`` with a residual (h is the next residual); both
    new tensors of x's dtype.  ``weight`` is ``[width]`` in x's dtype or fp32
    (None: ones).  y is computed from the unrounded sum; h is rounded once.
    Differentiable in x, weight and residual; the weight's gradient is summed
    over the rows in fp32 in a fixed order.  A row that holds an infinity or a
    NaN gives NaN where it stands, as the formula does.
    """
    if _eager(x):
        got = native().rms_norm(x, weight, residual, eps)
        if got is not None:
            return got
    _refuse_transforms("fused_rms_norm", x, weight, residual)
    _check(x, weight, residual, eps)
    if _needs_grad(x, weight, residual):
        return _RMSNormFn.apply(x, weight, residual, eps)
    y, _, *h = torch.ops.mlpk.rms_norm(x, weight, residual, eps)
    return (y, h[0]) if h else y


def fused_rms_norm_fp8(x: Tensor, weight: Optional[Tensor] = None, *, residual: Optional[Tensor] = None,
                       eps: float = 1e-6, group: int = 0):
    """The norm with an 8-bit output: ``(q, scale)``, or ``(q, scale, h)`` with a
    residual; ``q.float() * scale`` (each scale over its columns) is y.

    ``q`` is float8_e4m3fn of x's shape, ``scale`` fp32 ``[..., groups]``:
    max|y| / 448 over the row (``group=0``) or over each 128 columns
    (``group=128``, the last group may be shorter).  A NaN makes its group's
    scale NaN.  For inference: raises where a gradient would be needed.
    """
    if _eager(x):
        got = native().rms_norm_fp8(x, weight, residual, eps, group)
        if got is not None:
            return got
    _refuse_transforms("fused_rms_norm_fp8", x, weight, residual)
    _check(x, weight, residual, eps)
    _check_group(group)
    if _needs_grad(x, weight, residual):
        raise RuntimeError("fused_rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    return tuple(torch.ops.mlpk.rms_norm_fp8(x, weight, residual, eps, group))


class FusedRMSNorm(nn.Module):
    """RMS norm with a learned weight ``[width]``, initialised to ones."""

    def __init__(self, width: int, eps: float = 1e-6):
        super().__init__()
        if not 1 <= width <= _lib.NORM_MAX_WIDTH:
            raise ValueError(f"the width must be 1 to {_lib.NORM_MAX_WIDTH}, got {width}")
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(width))

    def forward(self, x, residual=None):
        return fused_rms_norm(x, self.weight, residual=residual, eps=self.eps)
