"""The feed-forward operators under tracers, dispatch modes, torch.compile and
torch.func: what is recorded are the operators, tangents and transforms are
refused, and a derivative of a gradient raises."""
import contextlib

import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from mlp_megakernel_b200 import FusedGatedMLP, FusedLinear, fp8_checkpoint, fp8_restore, fused_gated_mlp, fused_linear

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


class Recorder(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def randn(*shape, seed):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).bfloat16()


def inputs(seed, grad=False):
    shapes = ((30, 72), (72, 40), (40,), (30, 40), (72, 40), (40, 40))
    return [(randn(*s, seed=seed + i) * (0.2 if i else 1)).requires_grad_(grad) for i, s in enumerate(shapes)]


def linear(x, w, b, r, u, d):
    return fused_linear(x, w, b, activation="silu", residual=r), fused_linear(x, w)


def gated(x, w, b, r, u, d):
    return (fused_gated_mlp(x, w, u, d, residual=r),)


def checkpoint(x, w, b, r, u, d):
    q, scale = fp8_checkpoint(x)
    return q.float(), scale, fp8_restore(q, scale, torch.float16)


def linear_gradients(kept):
    def f(x, w, b, r, u, d):
        out = fused_linear(x, w, b, activation="gelu_tanh", residual=r, activation_dtype=kept)
        return torch.autograd.grad(out.float().square().sum(), (x, w, b, r))

    f.__name__ = f"linear_gradients{'_fp8' if kept else ''}"
    return f


def gated_gradients(kept):
    def f(x, w, b, r, u, d):
        out = fused_gated_mlp(x, w, u, d, residual=r, activation_dtype=kept)
        return torch.autograd.grad(out.float().square().sum(), (x, w, u, d, r))

    f.__name__ = f"gated_gradients{'_fp8' if kept else ''}"
    return f


FORWARDS = [linear, gated, checkpoint]
GRADIENTS = [f(kept) for kept in (None, FP8) for f in (linear_gradients, gated_gradients)]


def same(got, want):
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("f", FORWARDS + GRADIENTS)
def test_make_fx(f):
    grad = f in GRADIENTS
    graph = make_fx(f)(*inputs(1, grad))
    assert any(str(n.target).startswith("mlpk.") for n in graph.graph.nodes)
    same(graph(*inputs(21)), f(*inputs(21, grad)))


@pytest.mark.parametrize("f", FORWARDS)
def test_dispatch_mode_sees_the_operators(f):
    args = inputs(1)
    with Recorder() as mode:
        got = f(*args)
    assert any(name.startswith("mlpk.") for name in mode.seen)
    same(got, f(*args))


@pytest.mark.parametrize("f", GRADIENTS)
def test_backward_of_an_eager_graph_under_a_mode(f):
    args = inputs(1, True)
    if "linear" in f.__name__:
        out = fused_linear(*args[:3], activation="silu", activation_dtype=FP8 if "fp8" in f.__name__ else None)
        leaves, name = args[:3], "mlpk.linear_bwd"
    else:
        out = fused_gated_mlp(args[0], args[1], args[4], args[5], activation_dtype=FP8 if "fp8" in f.__name__ else None)
        leaves, name = [args[0], args[1], args[4], args[5]], "mlpk.gated_mlp_bwd"
    go = randn(*out.shape, seed=50)
    want = torch.autograd.grad(out, leaves, go, retain_graph=True)
    with Recorder() as mode:
        got = torch.autograd.grad(out, leaves, go, retain_graph=True)
    assert any(s.startswith(name) for s in mode.seen)
    same(got, want)


@pytest.mark.parametrize("kept", [None, FP8])
def test_compiled_modules(kept):
    torch.manual_seed(0)
    net = torch.nn.Sequential(FusedLinear(72, 40, activation="gelu_tanh", activation_dtype=kept),
                              FusedGatedMLP(40, 64, out_features=16, activation_dtype=kept)).cuda().bfloat16()
    compiled = torch.compile(net, fullgraph=True)
    x, go = randn(50, 72, seed=1), randn(50, 16, seed=2)
    outs, grads = [], []
    for f in (net, compiled):
        net.zero_grad()
        out = f(x)
        out.backward(go)
        outs.append(out.detach())
        grads.append([p.grad.clone() for p in net.parameters()])
    assert torch.equal(*outs)
    same(*grads)


def test_jit_trace():
    for f in FORWARDS:
        traced = torch.jit.trace(f, tuple(inputs(1)), check_trace=False)
        same(traced(*inputs(21)), f(*inputs(21)))


@pytest.mark.parametrize("needs_grad", [False, True])
def test_tangents_are_refused(needs_grad):
    x, w, b, r, u, d = inputs(1, needs_grad)

    def dual(t):
        return fwd.make_dual(t, torch.ones_like(t))

    with fwd.dual_level():
        for call in (lambda: fused_linear(dual(x), w), lambda: fused_linear(x, dual(w)), lambda: fused_linear(x, w, dual(b)),
                     lambda: fused_linear(x, w, residual=dual(r)), lambda: fused_gated_mlp(x, w, dual(u), d),
                     lambda: fused_gated_mlp(x, w, u, dual(d))):
            with pytest.raises(RuntimeError, match="forward"):
                call()
        if not needs_grad:
            with pytest.raises(RuntimeError, match="forward"):
                fp8_checkpoint(dual(x))
        same([fused_linear(x, w)], [fused_linear(x, w)])


def test_transforms_are_refused():
    x, w, b, r, u, d = inputs(1)
    for call in (lambda: torch.func.vmap(lambda t: fused_linear(t, w))(x[:, None]), lambda: torch.func.grad(lambda t: fused_linear(t, w).float().sum())(x),
                 lambda: torch.func.vmap(lambda t: fused_gated_mlp(t, w, u, d))(x[:, None]),
                 lambda: torch.func.vmap(lambda t: fp8_checkpoint(t)[1])(x[:, None])):
        with pytest.raises(RuntimeError, match="transform"):
            call()


@pytest.mark.parametrize("route", [contextlib.nullcontext, Recorder])
@pytest.mark.parametrize("which", range(4))
def test_a_derivative_of_a_gradient_raises(route, which):
    x, w, b, r, u, d = inputs(1, True)
    with route():
        out = [lambda: fused_linear(x, w), lambda: fused_linear(x, w, b, activation="silu"),
               lambda: fused_gated_mlp(x, w, u, d), lambda: fused_gated_mlp(x, w, u, d, activation_dtype=FP8)][which]()
    g, = torch.autograd.grad(out.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate|backward"):
        (g.float().square().sum() + sum(t.float().square().sum() for t in (x, w, u, d))).backward()


def test_nothing_raises_where_the_derivative_is_zero():
    """dw of one product does not depend on w, nor w_down's gradient on w_down: a penalty on it has no derivative."""
    x, w, b, r, u, d = inputs(1)
    for leaf, f in ((w, lambda t: fused_linear(x, t)), (d, lambda t: fused_gated_mlp(x, w, u, t)), (u, lambda t: fused_gated_mlp(x, w, t, d))):
        t = leaf.clone().requires_grad_()
        g, = torch.autograd.grad(f(t).float().sum(), t, create_graph=True)
        assert not g.requires_grad
