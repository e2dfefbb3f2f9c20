"""Derivatives of the block operators' gradients, which they do not have: where
one is asked for the backward raises; nothing is left out in silence, and nothing
raises where the derivative is truly zero."""
import contextlib

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from mlp_megakernel_b200 import expert_combine, expert_dispatch, expert_sort, fused_rms_norm

pytestmark = pytest.mark.gpu


def randn(*shape, seed):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


class PassOn(TorchDispatchMode):
    """Changes nothing; the calls under it are the operators of torch.ops.mlpk."""

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.fixture(params=["native", "operators"])
def route(request):
    """Both ways that a call takes: its context."""
    return contextlib.nullcontext if request.param == "native" else PassOn


def leaves():
    x, w, r = randn(12, 40, seed=1), randn(40, seed=2), randn(12, 40, seed=3)
    return x, w, r


def plan_and_rows():
    plan = expert_sort(torch.arange(24, device="cuda").view(12, 2) % 5 - 1, 4)  # some dropped
    return plan, randn(24, 40, seed=4), torch.rand(12, 2, device="cuda")


@pytest.mark.parametrize("wrt", ["x", "w", "r"])
@pytest.mark.parametrize("upstream", ["constant", "differentiable"])
def test_gradient_of_a_norms_gradient_raises(route, wrt, upstream):
    x, w, r = (t.requires_grad_() for t in leaves())
    with route():
        y, _ = fused_rms_norm(x, w, residual=r)
    leaf = {"x": x, "w": w, "r": r}[wrt]
    loss = y.sum() if upstream == "constant" else y.square().sum()
    g, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate|backward"):
        (g.square().sum() + x.square().sum() + w.square().sum() + r.square().sum()).backward()


def test_gradient_of_a_penalty_on_one_input_raises(route):
    x = leaves()[0].requires_grad_()
    with route():
        y = fused_rms_norm(x)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate|backward"):
        (g.norm() + x.square().sum()).backward()


@pytest.mark.parametrize("wrt", ["y", "weights"])
@pytest.mark.parametrize("upstream", ["constant", "differentiable"])
def test_gradient_of_a_combines_gradient_raises(route, wrt, upstream):
    plan, y, weights = plan_and_rows()
    y.requires_grad_()
    weights.requires_grad_()
    with route():
        out = expert_combine(y, weights, plan)
    loss = out.sum() if upstream == "constant" else out.square().sum()
    g, = torch.autograd.grad(loss, y if wrt == "y" else weights, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate|backward"):
        (g.square().sum() + y.square().sum() + weights.square().sum()).backward()


def test_gradient_of_a_dispatchs_gradient_raises(route):
    plan, _, _ = plan_and_rows()
    x = leaves()[0].requires_grad_()
    with route():
        rows = expert_dispatch(x, plan)
    g, = torch.autograd.grad(rows.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate|backward"):
        g.square().sum().backward()


def test_gradients_that_do_not_depend_on_anything(route):
    """Linear in what they are taken for, with a constant upstream gradient: a
    term with such a gradient adds nothing to the other terms' gradients."""
    plan, y, weights = plan_and_rows()
    x, w, r = leaves()
    for leaf, call in ((x, lambda t: expert_dispatch(t, plan)), (y, lambda t: expert_combine(t, weights, plan)),
                       (weights, lambda t: expert_combine(y, t, plan)), (w, lambda t: fused_rms_norm(x, t)),
                       (r, lambda t: fused_rms_norm(x, w, residual=t)[1])):
        leaf = leaf.clone().requires_grad_()
        with route():
            out = call(leaf)
        g, = torch.autograd.grad(out.sum(), leaf, create_graph=True)
        (g.square().sum() + leaf.square().sum()).backward()
        assert torch.equal(leaf.grad, 2 * leaf.detach())


def test_the_sum_of_the_norm_can_be_differentiated_twice(route):
    """h alone: its gradient passes the norm by, and has its own derivative."""
    x, w, r = (t.requires_grad_() for t in leaves())
    with route():
        _, h = fused_rms_norm(x, w, residual=r)
    g, = torch.autograd.grad(h.square().sum(), x, create_graph=True)
    again, = torch.autograd.grad(g.square().sum(), x)
    assert torch.allclose(again, 8 * (x + r).detach(), rtol=1e-6)


def test_plain_backward_with_create_graph_has_its_values(route):
    x, w, r = (t.requires_grad_() for t in leaves())
    plain = torch.autograd.grad(fused_rms_norm(x, w, residual=r)[0].square().sum(), (x, w, r))
    with route():
        y, _ = fused_rms_norm(x, w, residual=r)
    graph = torch.autograd.grad(y.square().sum(), (x, w, r), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, graph))
