"""The fused MLP's functional forward under tracers and dispatch modes that see
plain tensors: a recorded graph computes it on other inputs."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from mlp_megakernel_b200 import fused_mlp_fwd

pytestmark = pytest.mark.gpu


def inputs(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(*s, device="cuda", generator=g) * 0.1).half() for s in ((300, 128), (128, 128), (128, 128), (128, 128))]


def into(x, *weights):
    out = torch.zeros(x.shape[0], weights[-1].shape[1], device=x.device, dtype=x.dtype)
    fused_mlp_fwd(x, *weights, out=out)
    return out


@pytest.mark.parametrize("f", [fused_mlp_fwd, into])
def test_make_fx(f):
    graph = make_fx(f)(*inputs(1))
    assert any(str(n.target).startswith("mlpk.") for n in graph.graph.nodes)
    assert torch.equal(graph(*inputs(2)), f(*inputs(2)))


@pytest.mark.parametrize("f", [fused_mlp_fwd, into])
def test_jit_trace(f):
    traced = torch.jit.trace(f, tuple(inputs(1)), check_trace=False)
    assert torch.equal(traced(*inputs(2)), f(*inputs(2)))


def test_dispatch_mode():
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    with Mode():
        got = fused_mlp_fwd(*inputs(1))
    assert any(s.startswith("mlpk.fwd") for s in seen) and torch.equal(got, fused_mlp_fwd(*inputs(1)))
