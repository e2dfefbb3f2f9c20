"""Forward-mode derivatives and torch.func's transforms, which the block operators
do not have: a call that would need one raises in the operators' own words; none
drops a tangent in silence, and tensors that are not concerned go on."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.utils._python_dispatch import TorchDispatchMode

from mlp_megakernel_b200 import expert_combine, expert_dispatch, expert_sort, fused_rms_norm, fused_rms_norm_fp8

pytestmark = pytest.mark.gpu


class PassOn(TorchDispatchMode):
    """Changes nothing; the calls under it are the operators of torch.ops.mlpk."""

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def randn(*shape, seed):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def leaves():
    return randn(12, 40, seed=1), randn(40, seed=2), randn(12, 40, seed=3)


def plan_and_rows():
    plan = expert_sort(torch.arange(24, device="cuda").view(12, 2) % 5 - 1, 4)  # some dropped
    return plan, randn(24, 40, seed=4), torch.rand(12, 2, device="cuda")


@pytest.mark.parametrize("needs_grad", [False, True])
def test_tangents_are_refused(needs_grad):
    x, w, r = leaves()
    plan, y, weights = plan_and_rows()

    def dual(t):
        return fwd.make_dual(t.clone().requires_grad_(needs_grad), torch.ones_like(t))

    with fwd.dual_level():
        calls = [lambda: fused_rms_norm(dual(x)), lambda: fused_rms_norm(x, dual(w)),
                 lambda: fused_rms_norm(x, residual=dual(r)), lambda: expert_dispatch(dual(x), plan),
                 lambda: expert_combine(dual(y), weights, plan), lambda: expert_combine(y, dual(weights), plan)]
        if not needs_grad:
            calls.append(lambda: fused_rms_norm_fp8(dual(x)))
        for call in calls:
            with pytest.raises(RuntimeError, match="forward"):
                call()
        # other tensors of the same program may have tangents
        assert torch.equal(fused_rms_norm(x, w), fused_rms_norm(x, w))


@pytest.mark.parametrize("route", [contextlib.nullcontext, PassOn])
def test_tangents_of_upstream_gradients_are_refused(route):
    x, w, _ = leaves()
    plan, y, weights = plan_and_rows()
    x.requires_grad_()
    y.requires_grad_()
    with route():
        outputs = [(fused_rms_norm(x, w), x), (expert_dispatch(x, plan), x), (expert_combine(y, weights, plan), y)]
    for out, leaf in outputs:
        with fwd.dual_level():
            g = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward"):
                torch.autograd.grad(out, leaf, g, retain_graph=True)
        torch.autograd.grad(out, leaf, torch.ones_like(out))


def test_function_transforms_are_refused():
    """In the operators' own words, not by an error about a pointer."""
    x, w, r = leaves()
    plan, rows, weights = plan_and_rows()
    for f in (lambda t: fused_rms_norm(t, w), lambda t: fused_rms_norm_fp8(t, w)[1],
              lambda t: fused_rms_norm(x, residual=t.expand_as(x))[0]):
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.func.vmap(f)(x)
    for f in (lambda t: fused_rms_norm(t, w).float().sum(), lambda t: expert_dispatch(t, plan).float().sum()):
        with pytest.raises(RuntimeError, match="torch.func"):
            torch.func.grad(f)(x)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.grad(lambda t: expert_combine(rows, t, plan).float().sum())(weights)
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.vmap(lambda i: expert_sort(i, 5).row_of)(torch.zeros(4, 30, 2, device="cuda", dtype=torch.int64))
    # tensors that the transform does not touch are as always
    got = torch.func.vmap(lambda t: t + fused_rms_norm(x, w)[0])(x)
    assert torch.equal(got, x + fused_rms_norm(x, w)[0])
