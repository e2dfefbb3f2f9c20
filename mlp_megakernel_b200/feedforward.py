"""Feed-forward layers of any width on tensor cores, and activations kept in
8 bits (no counterpart in the reference, whose layers are at most 256 wide and
have one activation).

* ``fused_linear(x, weight, bias, activation=, residual=)`` -- one matrix product
  with bias, activation and residual in its epilogue;
* ``fused_gated_mlp(x, w_gate, w_up, w_down, activation=, residual=)`` -- both
  projections of a gated block, the activation and the product in one kernel,
  the projection back with the residual in a second;
* ``fp8_checkpoint(x)`` / ``fp8_restore(q, scale, dtype)`` -- values kept in 8
  bits with a power-of-two scale for each row and 128 columns, and back;
* ``FusedLinear``, ``FusedGatedMLP`` -- the modules.

Operands are fp16 or bf16, accumulators and everything in an epilogue fp32.  The
products are differentiable; ``activation_dtype=torch.float8_e4m3fn`` keeps what
their backward needs (the input, the values before the activation) as such
checkpoints instead of in the operands' type.  Weights are ``[in, out]``, or the
transpose of a contiguous ``[out, in]``, read where they are.  Widths are
multiples of 8.  The kernels run on the current CUDA stream; there is no CPU
path.  Eager calls go through the native binding (_native.py); under
torch.compile, tracers and dispatch modes and on fake tensors the calls are the
operators ``torch.ops.mlpk.linear`` / ``linear_bwd`` / ``gated_mlp`` /
``gated_mlp_bwd`` / ``fp8_checkpoint`` / ``fp8_restore``.
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor

from . import _lib
from ._native import native
from .norm import DTYPES, _eager, _needs_grad, _refuse_transforms

FP8 = torch.float8_e4m3fn
ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu_tanh": 3, "softplus": 4, "sigmoid": 5}
_OPERANDS = (torch.float16, torch.bfloat16)


# ------------------------------------------------------------ checks
def _act_code(activation) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def _check_act(act) -> None:
    if not 0 <= act <= 5:
        raise ValueError(f"there is no activation {act}")


def _keeps_fp8(activation_dtype, dtype) -> bool:
    if activation_dtype == dtype:
        return False
    _check_kept_type(activation_dtype)
    return activation_dtype is not None


def _check_kept_type(activation_dtype) -> None:
    if activation_dtype not in (None, FP8):
        raise TypeError(f"activation_dtype must be None (the operands' type) or {FP8}, got {activation_dtype}")


def _require_cuda(t) -> None:
    if isinstance(t, Tensor) and not t.is_cuda:
        raise RuntimeError("the feed-forward operators run on CUDA (sm_100) only; got a CPU tensor")


def _check_x(x, what="x") -> None:
    if not isinstance(x, Tensor) or x.dim() < 1:
        raise ValueError(f"{what} must be a tensor [..., width]")
    if x.dtype not in _OPERANDS:
        raise TypeError(f"{what} must be fp16 or bf16, got {x.dtype}")
    _check_width(x.shape[-1])
    if x.numel() // x.shape[-1] > _lib.FF_MAX_ROWS:
        raise ValueError(f"{what} has more than {_lib.FF_MAX_ROWS} rows")


def _check_width(width) -> None:
    if width < 8 or width % 8 or width > _lib.FF_MAX_WIDTH:
        raise ValueError(f"widths must be multiples of 8 up to {_lib.FF_MAX_WIDTH}, got {width}")


def _check_weight(what, w, d_in, x, d_out=None) -> None:
    if not isinstance(w, Tensor) or w.dim() != 2 or w.shape[0] != d_in or w.dtype != x.dtype or w.device != x.device \
            or (d_out is not None and w.shape[1] != d_out):
        raise ValueError(f"{what} must be a [{d_in}, {'width' if d_out is None else d_out}] tensor of {x.dtype} on {x.device}")
    _check_width(w.shape[1])


def _check_residual(residual, x, d_out) -> None:
    shape = (*x.shape[:-1], d_out)
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual must be a {shape} {x.dtype} tensor on {x.device}")


def _check_linear(x, weight, bias, residual) -> None:
    _check_x(x)
    _check_weight("weight", weight, x.shape[-1], x)
    n = weight.shape[1]
    if bias is not None and (bias.shape != (n,) or bias.device != x.device
                             or (bias.dtype != x.dtype and bias.dtype != torch.float32)):
        raise ValueError(f"bias must be a [{n}] tensor of {x.dtype} or float32 on {x.device}")
    _check_residual(residual, x, n)


def _check_gated(x, w_gate, w_up, w_down, residual) -> None:
    _check_x(x)
    _check_weight("w_gate", w_gate, x.shape[-1], x)
    _check_weight("w_up", w_up, x.shape[-1], x, w_gate.shape[1])
    _check_weight("w_down", w_down, w_gate.shape[1], x)
    _check_residual(residual, x, w_down.shape[1])


def _check_keep(keep) -> None:
    if keep not in (0, 1, 2):
        raise ValueError(f"keep must be 0, 1 (the operands' type) or 2 (8 bits), got {keep}")


def _pitch(width) -> int:
    return -(-width // 128) * 128


def _check_kept(what, t, scale, rows, width, ref) -> None:
    """What a forward kept: values of ref's type, or 8-bit ones with their scales."""
    if t.dtype == ref.dtype:
        ok = t.shape == (rows, width) and scale is None
    else:
        ok = t.dtype == FP8 and t.shape == (rows, _pitch(width)) and scale is not None and \
            scale.shape == (rows, -(-width // 128)) and scale.dtype == torch.float32 and scale.device == ref.device
    if not ok or t.device != ref.device or not t.is_contiguous() or (scale is not None and not scale.is_contiguous()):
        raise ValueError(f"{what} must be what the forward kept")


def _check_saved_x(x, x_scale, ref, width) -> None:
    """The input, or its checkpoint; rows of `ref`'s."""
    if x.dim() < 1 or x.shape[-1] != width or x.numel() // width != ref.numel() // ref.shape[-1] or x.device != ref.device:
        raise ValueError("x must be the forward's input")
    if x_scale is None:
        if x.dtype != ref.dtype:
            raise ValueError("x must be the forward's input")
    else:
        _check_quantized(x, x_scale)


def _check_linear_bwd(grad_out, x, x_scale, weight, z, z_scale, act, db_dtype, want) -> None:
    _check_act(act)
    _check_x(grad_out, "grad_out")
    rows, n = grad_out.numel() // grad_out.shape[-1], grad_out.shape[-1]
    if weight.dim() != 2 or weight.shape[1] != n or weight.dtype != grad_out.dtype or weight.device != grad_out.device:
        raise ValueError(f"weight must be a [width, {n}] tensor of {grad_out.dtype} on {grad_out.device}")
    _check_width(weight.shape[0])
    if act and (z is None):
        raise ValueError("z is missing: the activation's derivative needs it")
    if act:
        _check_kept("z", z, z_scale, rows, n, grad_out)
    if want[1]:
        if x is None:
            raise ValueError("x is missing: the weight's gradient needs it")
        _check_saved_x(x, x_scale, grad_out, weight.shape[0])
    if want[2] and db_dtype not in (grad_out.dtype, torch.float32):
        raise ValueError(f"the bias gradient must be {grad_out.dtype} or float32")


def _check_gated_bwd(grad_out, x, x_scale, w_gate, w_up, w_down, g, g_scale, u, u_scale, act, want) -> None:
    _check_act(act)
    _check_x(grad_out, "grad_out")
    rows = grad_out.numel() // grad_out.shape[-1]
    h = w_down.shape[0]
    _check_weight("w_down", w_down, h, grad_out, grad_out.shape[-1])
    _check_width(h)
    _check_width(w_gate.shape[0])
    _check_weight("w_gate", w_gate, w_gate.shape[0], grad_out, h)
    _check_weight("w_up", w_up, w_gate.shape[0], grad_out, h)
    _check_kept("g", g, g_scale, rows, h, grad_out)
    _check_kept("u", u, u_scale, rows, h, grad_out)
    if g.dtype != u.dtype:
        raise ValueError("g and u must be kept alike")
    if want[1]:
        if x is None:
            raise ValueError("x is missing: the weights' gradients need it")
        _check_saved_x(x, x_scale, grad_out, w_gate.shape[0])


def _check_columns(x) -> None:
    if x.shape[-1] > _lib.FP8_MAX_WIDTH:  # the C calls' int
        raise ValueError(f"rows must have at most {_lib.FP8_MAX_WIDTH} columns, got {x.shape[-1]}: view them as more rows")


def _check_values(x) -> None:
    if not isinstance(x, Tensor) or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be a tensor [..., width]")
    if x.dtype not in DTYPES:
        raise TypeError(f"fp8_checkpoint takes fp16, bf16 or fp32, got {x.dtype}")
    _check_columns(x)


def _check_quantized(q, scale) -> None:
    if not isinstance(q, Tensor) or q.dim() < 1 or q.shape[-1] < 1 or q.dtype != FP8:
        raise ValueError(f"q must be a {FP8} tensor [..., width]")
    _check_columns(q)
    want = (*q.shape[:-1], -(-q.shape[-1] // 128))
    if not isinstance(scale, Tensor) or scale.shape != want or scale.dtype != torch.float32 or scale.device != q.device:
        raise ValueError(f"scale must be a {want} float32 tensor on {q.device}")


# ------------------------------------------------------------ torch.ops.mlpk
def _kept_fake(ref, rows, width, keep):
    """[values] or [values, scales] as a forward keeps them."""
    if keep == 2:
        return [ref.new_empty((rows, _pitch(width)), dtype=FP8), ref.new_empty((rows, -(-width // 128)), dtype=torch.float32)]
    return [ref.new_empty((rows, width))] if keep else []


@torch.library.custom_op("mlpk::linear", mutates_args=())
def _linear_op(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor], act: int,
               keep: int) -> list[Tensor]:
    """[out], and z (with its scales) as `keep` says: 0 not, 1 in x's type, 2 in 8 bits."""
    _require_cuda(x)
    _check_linear(x, weight, bias, residual)
    _check_act(act)
    _check_keep(keep)
    return [t for t in native().linear_forward(x, weight, bias, residual, act, keep) if t is not None]


@_linear_op.register_fake
def _linear_fake(x, weight, bias, residual, act, keep):
    _check_linear(x, weight, bias, residual)
    _check_act(act)
    _check_keep(keep)
    n = weight.shape[1]
    return [x.new_empty((*x.shape[:-1], n))] + _kept_fake(x, x.numel() // x.shape[-1], n, keep)


def _dw_fake(w):
    """A weight's gradient, in its layout."""
    k, n = w.shape
    return w.new_empty((n, k)).t() if not w.is_contiguous() and w.t().is_contiguous() else w.new_empty((k, n))


@torch.library.custom_op("mlpk::linear_bwd", mutates_args=())
def _linear_bwd_op(grad_out: Tensor, x: Optional[Tensor], x_scale: Optional[Tensor], weight: Tensor, z: Optional[Tensor],
                   z_scale: Optional[Tensor], act: int, db_dtype: torch.dtype, want_dx: bool, want_dw: bool,
                   want_db: bool) -> list[Tensor]:
    """[dx], [dw] and [db], as wanted.  x with x_scale: its checkpoint."""
    _require_cuda(grad_out)
    _check_linear_bwd(grad_out, x, x_scale, weight, z, z_scale, act, db_dtype, (want_dx, want_dw, want_db))
    got = native().linear_backward(grad_out, x, x_scale, weight, z, z_scale, act, db_dtype == torch.float32, want_dx,
                                   want_dw, want_db)
    return [t for t in got if t is not None]


@_linear_bwd_op.register_fake
def _linear_bwd_fake(grad_out, x, x_scale, weight, z, z_scale, act, db_dtype, want_dx, want_dw, want_db):
    _check_linear_bwd(grad_out, x, x_scale, weight, z, z_scale, act, db_dtype, (want_dx, want_dw, want_db))
    k, n = weight.shape
    return ([grad_out.new_empty((*grad_out.shape[:-1], k))] if want_dx else []) + ([_dw_fake(weight)] if want_dw else []) + \
        ([grad_out.new_empty((n,), dtype=db_dtype)] if want_db else [])


@torch.library.custom_op("mlpk::gated_mlp", mutates_args=())
def _gated_op(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, residual: Optional[Tensor], act: int,
              keep: int) -> list[Tensor]:
    """[out], and g (with its scales) and u (with its) as `keep` says."""
    _require_cuda(x)
    _check_gated(x, w_gate, w_up, w_down, residual)
    _check_act(act)
    _check_keep(keep)
    return [t for t in native().gated_forward(x, w_gate, w_up, w_down, residual, act, keep) if t is not None]


@_gated_op.register_fake
def _gated_fake(x, w_gate, w_up, w_down, residual, act, keep):
    _check_gated(x, w_gate, w_up, w_down, residual)
    _check_act(act)
    _check_keep(keep)
    rows, h = x.numel() // x.shape[-1], w_gate.shape[1]
    return [x.new_empty((*x.shape[:-1], w_down.shape[1])), *_kept_fake(x, rows, h, keep), *_kept_fake(x, rows, h, keep)]


@torch.library.custom_op("mlpk::gated_mlp_bwd", mutates_args=())
def _gated_bwd_op(grad_out: Tensor, x: Optional[Tensor], x_scale: Optional[Tensor], w_gate: Tensor, w_up: Tensor,
                  w_down: Tensor, g: Tensor, g_scale: Optional[Tensor], u: Tensor, u_scale: Optional[Tensor], act: int,
                  want_dx: bool, want_dgu: bool, want_dd: bool) -> list[Tensor]:
    """[dx], [dw_gate, dw_up] and [dw_down], as wanted."""
    _require_cuda(grad_out)
    _check_gated_bwd(grad_out, x, x_scale, w_gate, w_up, w_down, g, g_scale, u, u_scale, act, (want_dx, want_dgu, want_dd))
    got = native().gated_backward(grad_out, x, x_scale, w_gate, w_up, w_down, g, g_scale, u, u_scale, act, want_dx,
                                  want_dgu, want_dd)
    return [t for t in got if t is not None]


@_gated_bwd_op.register_fake
def _gated_bwd_fake(grad_out, x, x_scale, w_gate, w_up, w_down, g, g_scale, u, u_scale, act, want_dx, want_dgu, want_dd):
    _check_gated_bwd(grad_out, x, x_scale, w_gate, w_up, w_down, g, g_scale, u, u_scale, act, (want_dx, want_dgu, want_dd))
    alike = _dw_fake(w_gate).stride() == _dw_fake(w_up).stride()
    both = [_dw_fake(w) if alike else w.new_empty(w.shape) for w in (w_gate, w_up)]
    return ([grad_out.new_empty((*grad_out.shape[:-1], w_gate.shape[0]))] if want_dx else []) + \
        (both if want_dgu else []) + ([_dw_fake(w_down)] if want_dd else [])


@torch.library.custom_op("mlpk::fp8_checkpoint", mutates_args=())
def _checkpoint_op(x: Tensor) -> list[Tensor]:
    """[q, scale]."""
    _require_cuda(x)
    _check_values(x)
    return list(native().checkpoint(x))


@_checkpoint_op.register_fake
def _checkpoint_fake(x):
    _check_values(x)
    return [x.new_empty(x.shape, dtype=FP8), x.new_empty((*x.shape[:-1], -(-x.shape[-1] // 128)), dtype=torch.float32)]


@torch.library.custom_op("mlpk::fp8_restore", mutates_args=())
def _restore_op(q: Tensor, scale: Tensor, dtype: torch.dtype) -> Tensor:
    _require_cuda(q)
    _check_quantized(q, scale)
    _check_restored(dtype)
    return native().restore(q, scale, dtype)


@_restore_op.register_fake
def _restore_fake(q, scale, dtype):
    _check_quantized(q, scale)
    _check_restored(dtype)
    return q.new_empty(q.shape, dtype=dtype)


def _check_restored(dtype) -> None:
    if dtype not in DTYPES:
        raise TypeError(f"fp8_restore gives fp16, bf16 or fp32, not {dtype}")


# ------------------------------------------------------------ autograd
def _checkpoint_of(x, fp8):
    """What a node keeps of its input: (x, None) or its checkpoint."""
    return torch.ops.mlpk.fp8_checkpoint(x) if fp8 else (x, None)


class _LinearFn(torch.autograd.Function):
    """The node that tracers and modes see (as _GatedFn).  Its gradients are
    operators without a derivative: asking for one raises."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, fp8):
        wanted = ctx.needs_input_grad
        keep = (2 if fp8 else 1) if act and any(wanted[:3]) else 0
        out, *z = torch.ops.mlpk.linear(x, weight, bias, residual, act, keep)
        kept = _checkpoint_of(x, fp8) if wanted[1] else (None, None)
        ctx.act, ctx.db_dtype = act, x.dtype if bias is None else bias.dtype
        ctx.save_for_backward(*kept, weight, *(z + [None] * (2 - len(z))))
        return out

    @staticmethod
    def backward(ctx, grad):
        x, x_scale, weight, z, z_scale = ctx.saved_tensors
        _refuse_transforms("the gradient of fused_linear", grad, x, weight)
        want = ctx.needs_input_grad
        got = []
        if any(want[:3]):
            got = torch.ops.mlpk.linear_bwd(grad, x, x_scale, weight, z, z_scale, ctx.act, ctx.db_dtype, *want[:3])
        got = iter(got)
        grads = [next(got) if w else None for w in want[:3]]
        return *grads, grad if want[3] else None, None, None


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, residual, act, fp8):
        wanted = ctx.needs_input_grad
        keep = (2 if fp8 else 1) if any(wanted[:4]) else 0
        out, *kept = torch.ops.mlpk.gated_mlp(x, w_gate, w_up, w_down, residual, act, keep)
        g, g_scale, u, u_scale = kept if keep == 2 else (kept[0], None, kept[1], None) if keep else (None,) * 4
        ctx.act = act
        ctx.save_for_backward(*(_checkpoint_of(x, fp8) if wanted[1] or wanted[2] else (None, None)), w_gate, w_up, w_down,
                              g, g_scale, u, u_scale)
        return out

    @staticmethod
    def backward(ctx, grad):
        saved = ctx.saved_tensors
        _refuse_transforms("the gradient of fused_gated_mlp", grad, *saved)
        dx, dg, du, dd, dr, *_ = ctx.needs_input_grad
        grads = [None] * 4
        if dx or dg or du or dd:
            got = iter(torch.ops.mlpk.gated_mlp_bwd(grad, *saved, ctx.act, dx, dg or du, dd))
            grads[0] = next(got) if dx else None
            both = (next(got), next(got)) if dg or du else (None, None)
            grads[1], grads[2] = both[0] if dg else None, both[1] if du else None
            grads[3] = next(got) if dd else None
        return *grads, grad if dr else None, None, None


# ------------------------------------------------------------ public calls
def fused_linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, *, activation: Optional[str] = None,
                 residual: Optional[Tensor] = None, activation_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``activation(x @ weight + bias) + residual``, a new ``[..., out]`` tensor.

    ``x`` is fp16 or bf16 ``[..., in]``, ``weight`` ``[in, out]`` of its type
    (contiguous, or the transpose of a contiguous tensor), ``bias`` ``[out]`` of
    its type or fp32, ``residual`` as the output.  ``activation`` is None,
    "relu", "silu", "gelu_tanh", "softplus" or "sigmoid".  Accumulation and all
    of the epilogue are fp32, rounded once.  Differentiable in all four; the
    weight's and the bias's gradients are summed over the rows in fp32 in a fixed
    order.  ``activation_dtype`` is the precision of what the backward keeps (x
    where the weight needs a gradient, the values before the activation): x's
    type, or ``torch.float8_e4m3fn`` (fp8_checkpoint).  In x's type a finite value
    beyond its largest (65504 in fp16) is kept as that; the gradients are the same,
    since every derivative is constant out there.
    """
    act = _act_code(activation)
    fp8 = _keeps_fp8(activation_dtype, getattr(x, "dtype", None))
    if _eager(x):
        got = native().linear(x, weight, bias, residual, act, fp8)
        if got is not None:
            return got
    _refuse_transforms("fused_linear", x, weight, bias, residual)
    _require_cuda(x)
    _check_linear(x, weight, bias, residual)
    if _needs_grad(x, weight, bias, residual):
        return _LinearFn.apply(x, weight, bias, residual, act, fp8)
    return torch.ops.mlpk.linear(x, weight, bias, residual, act, 0)[0]


def fused_gated_mlp(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, *, activation: Optional[str] = "silu",
                    residual: Optional[Tensor] = None, activation_dtype: Optional[torch.dtype] = None) -> Tensor:
    """``(activation(x @ w_gate) * (x @ w_up)) @ w_down + residual``.

    ``x`` is fp16 or bf16 ``[..., in]``, ``w_gate`` and ``w_up`` ``[in, hidden]``,
    ``w_down`` ``[hidden, out]`` of its type (each contiguous or the transpose of
    a contiguous tensor), ``residual`` ``[..., out]``.  Two products; the hidden
    values are rounded to x's type between them.  Differentiable in all of them:
    the backward forms both hidden gradients and the hidden values again in the
    epilogue of one product.  ``activation`` and ``activation_dtype`` as in
    fused_linear (kept: x, and both projections).  Where a projection is beyond the
    largest value of x's type (65504 in fp16), the gradients are those of a
    projection of that value; kept in 8 bits it stays within 1/16 of itself.
    """
    act = _act_code(activation)
    fp8 = _keeps_fp8(activation_dtype, getattr(x, "dtype", None))
    if _eager(x):
        got = native().gated_mlp(x, w_gate, w_up, w_down, residual, act, fp8)
        if got is not None:
            return got
    _refuse_transforms("fused_gated_mlp", x, w_gate, w_up, w_down, residual)
    _require_cuda(x)
    _check_gated(x, w_gate, w_up, w_down, residual)
    if _needs_grad(x, w_gate, w_up, w_down, residual):
        return _GatedFn.apply(x, w_gate, w_up, w_down, residual, act, fp8)
    return torch.ops.mlpk.gated_mlp(x, w_gate, w_up, w_down, residual, act, 0)[0]


def fp8_checkpoint(x: Tensor):
    """``(q, scale)``: x in 8 bits, for a backward pass or a cache of the caller's.

    ``x`` is fp16, bf16 or fp32 ``[..., width]`` of any width below 2^31; ``q`` is
    float8_e4m3fn of its shape, ``scale`` fp32 ``[..., ceil(width / 128)]``: the
    smallest power of two (2^-126 at least) with ``max|x| / scale <= 448`` over
    its 128 columns, NaN where one of them is not finite.  A value is off by 1/16
    of itself at most (scale / 1024 for the smallest).  Raises where a gradient
    would be needed.
    """
    if _eager(x):
        got = native().fp8_checkpoint(x)
        if got is not None:
            return got
    _refuse_transforms("fp8_checkpoint", x)
    _require_cuda(x)
    _check_values(x)
    if _needs_grad(x):
        raise RuntimeError("fp8_checkpoint has no gradient: call it under torch.no_grad()")
    return tuple(torch.ops.mlpk.fp8_checkpoint(x))


def fp8_restore(q: Tensor, scale: Tensor, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``q * scale`` (each scale over its 128 columns) as fp16, bf16 or fp32: exact
    in bf16 and fp32, and in fp16 within its range; a finite product beyond the
    type's largest value becomes that value."""
    if _eager(q) and isinstance(scale, Tensor) and dtype in DTYPES:
        got = native().fp8_restore(q, scale, dtype)
        if got is not None:
            return got
    _refuse_transforms("fp8_restore", q, scale)
    _require_cuda(q)
    _check_quantized(q, scale)
    _check_restored(dtype)
    return torch.ops.mlpk.fp8_restore(q, scale, dtype)


# ------------------------------------------------------------ modules
def _uniform(*shape) -> nn.Parameter:
    bound = 1 / math.sqrt(shape[0])
    return nn.Parameter(torch.empty(*shape).uniform_(-bound, bound))


def _operand_type(x: Tensor) -> torch.dtype:
    """The type a module computes in: autocast's, else its input's."""
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype


class FusedLinear(nn.Module):
    """``activation(x @ weight + bias) + residual`` with ``weight`` ``[in, out]``.
    Parameters of another type (fp32 ones, say) are cast to x's, or autocast's; an
    fp32 bias is added as it is."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, activation: Optional[str] = None,
                 activation_dtype: Optional[torch.dtype] = None):
        super().__init__()
        _check_width(in_features)
        _check_width(out_features)
        _act_code(activation)
        _check_kept_type(activation_dtype)
        self.activation, self.activation_dtype = activation, activation_dtype
        self.weight = _uniform(in_features, out_features)
        self.bias = nn.Parameter(torch.zeros(out_features)) if bias else None

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        t = _operand_type(x)
        bias = self.bias if self.bias is None or self.bias.dtype == torch.float32 else self.bias.to(t)
        return fused_linear(x.to(t), self.weight.to(t), bias, activation=self.activation,
                            residual=None if residual is None else residual.to(t),
                            activation_dtype=self.activation_dtype)


class FusedGatedMLP(nn.Module):
    """A gated feed-forward block ``D -> H -> out_features`` (D if None):
    ``(activation(x @ w_gate) * (x @ w_up)) @ w_down + residual``."""

    def __init__(self, D: int, H: int, out_features: Optional[int] = None, activation: Optional[str] = "silu",
                 activation_dtype: Optional[torch.dtype] = None):
        super().__init__()
        out_features = D if out_features is None else out_features
        for width in (D, H, out_features):
            _check_width(width)
        _act_code(activation)
        _check_kept_type(activation_dtype)
        self.activation, self.activation_dtype = activation, activation_dtype
        self.w_gate, self.w_up, self.w_down = _uniform(D, H), _uniform(D, H), _uniform(H, out_features)

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        t = _operand_type(x)
        return fused_gated_mlp(x.to(t), self.w_gate.to(t), self.w_up.to(t), self.w_down.to(t), activation=self.activation,
                               residual=None if residual is None else residual.to(t),
                               activation_dtype=self.activation_dtype)
