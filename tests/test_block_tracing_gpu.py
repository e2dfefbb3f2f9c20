"""The block operators under tracers and dispatch modes that see plain tensors:
what they record has to be the operators, and a recorded graph has to compute
them on other inputs."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from mlp_megakernel_b200 import (ExpertPlan, FusedRMSNorm, expert_combine, expert_dispatch, expert_sort, fused_rms_norm,
                                 fused_rms_norm_fp8)

pytestmark = pytest.mark.gpu


class Recorder(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


def randn(*shape, seed):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).half()


def norm(x, w, r):
    y, h = fused_rms_norm(x, w, residual=r)
    return y, h, fused_rms_norm(x)


def norm_fp8(x, w, r):
    q, scale, h = fused_rms_norm_fp8(x, w, residual=r, group=128)
    return q.float(), scale, h


def norm_gradients(x, w, r):
    y, h = fused_rms_norm(x, w, residual=r)
    return torch.autograd.grad((y.float().square().sum(), h.float().sum()), (x, w, r))


def experts(x, w, r):
    ids = (x[:, :2].float() * 3).floor().long()
    plan = expert_sort(ids, 5)
    rows = expert_dispatch(x, plan)
    return plan.row_of, plan.offsets, rows, expert_combine(rows * 2, r[:, :2], plan)


def expert_gradients(x, w, r):
    ids = (x[:, :2].detach().float() * 3).floor().long()
    plan = expert_sort(ids, 5)
    weights = r[:, :2].float()
    out = expert_combine(expert_dispatch(x, plan), weights, plan)
    return torch.autograd.grad(out.float().square().sum(), (x, r))


def inputs(seed, grad):
    return [t.requires_grad_(grad) for t in (randn(30, 200, seed=seed), randn(200, seed=seed + 1), randn(30, 200, seed=seed + 2))]


FORWARDS, GRADIENTS = [norm, norm_fp8, experts], [norm_gradients, expert_gradients]


def same(got, want):
    assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("f", FORWARDS + GRADIENTS)
def test_make_fx(f):
    grad = f in GRADIENTS
    graph = make_fx(f)(*inputs(1, grad))
    assert any(str(n.target).startswith("mlpk.") for n in graph.graph.nodes)
    same(graph(*inputs(11, False)), f(*inputs(11, grad)))


@pytest.mark.parametrize("f", FORWARDS)
def test_jit_trace(f):
    with torch.no_grad():
        traced = torch.jit.trace(f, tuple(inputs(1, False)), check_trace=False)
        same(traced(*inputs(11, False)), f(*inputs(11, False)))


def test_jit_trace_of_the_module():
    m = FusedRMSNorm(200).cuda()
    traced = torch.jit.trace(m, (inputs(1, False)[0],), check_trace=False)
    x = inputs(11, False)[0]
    assert torch.equal(traced(x), m(x))


@pytest.mark.parametrize("f", FORWARDS)
def test_dispatch_mode_sees_the_operators(f):
    args = inputs(1, False)
    with Recorder() as mode:
        got = f(*args)
    assert any(name.startswith("mlpk.") for name in mode.seen)
    same(got, f(*args))


def outputs_and_leaves():
    """Outputs of calls before any mode, with what their gradients are for."""
    x, w, r = inputs(1, True)
    y, h = fused_rms_norm(x, w, residual=r)
    plan = expert_sort(torch.arange(60, device="cuda").view(30, 2) % 4 - 1, 3)
    rows = expert_dispatch(x, plan)
    weights = torch.rand(30, 2, device="cuda", requires_grad=True)
    out = expert_combine(rows.detach().requires_grad_(), weights, plan)
    return [((y, h), (x, w, r), "rms_norm_bwd"), ((y,), (x, w), "rms_norm_bwd"), ((rows,), (x,), "expert_combine"),
            ((out,), (weights,), "expert_combine_bwd")]


@pytest.mark.parametrize("case", range(4))
def test_backward_under_a_mode(case):
    """The graph was made before: its gradients are the operators too."""
    out, leaves, name = outputs_and_leaves()[case]
    grads = [randn(*o.shape, seed=20 + k).to(o.dtype) for k, o in enumerate(out)]
    want = torch.autograd.grad(out, leaves, grads, retain_graph=True)
    with Recorder() as mode:
        got = torch.autograd.grad(out, leaves, grads, retain_graph=True)
    assert any(s.startswith(f"mlpk.{name}.") for s in mode.seen)
    same(got, want)
    graph = make_fx(lambda *g: torch.autograd.grad(out, leaves, g, retain_graph=True))(*[torch.zeros_like(g) for g in grads])
    same(graph(*grads), want)


def test_plan_under_a_mode_is_a_plan():
    with Recorder():
        assert isinstance(expert_sort(torch.zeros(3, 2, device="cuda", dtype=torch.int32), 2), ExpertPlan)
