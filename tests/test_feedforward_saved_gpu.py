"""What autograd saves for the feed-forward operators may come back from a hook in another layout, or as a copy off the
16-byte grid: the gradients are the same bits.  Anything else that a hook gives back is refused before a kernel runs."""
import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

from mlp_megakernel_b200 import _lib, fused_gated_mlp, fused_linear

pytestmark = pytest.mark.gpu
F16, F32, FP8 = torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def status():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def randn(*shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(F16)


def bits(t):
    return t.view(torch.uint8) if t.dtype == FP8 else t


def columns(t):
    """The same values, the columns contiguous."""
    return bits(t).t().contiguous().t().view(t.dtype) if t.dtype == FP8 else t.t().contiguous().t()


def spread(t):
    """Every second column of a wider tensor."""
    wide = torch.zeros(t.shape[0], 2 * t.shape[1], device=t.device, dtype=bits(t).dtype)
    wide[:, ::2] = bits(t)
    return wide.view(t.dtype)[:, ::2]


def off(t):
    """A copy that begins one element past the grid."""
    flat = torch.empty(t.numel() + 1, device=t.device, dtype=bits(t).dtype)
    flat[1:] = bits(t).reshape(-1)
    return flat.view(t.dtype)[1:].view(t.shape)


def steps(kept):
    x, w, b = randn(40, 72, seed=1), randn(72, 264, seed=2, scale=0.1), randn(264, seed=3)
    wu, wd = randn(72, 264, seed=4, scale=0.1), randn(264, 136, seed=5, scale=0.1)
    a = [t.clone().requires_grad_() for t in (x, w, b)]
    c = [t.clone().requires_grad_() for t in (x, w, wu, wd)]
    yield lambda: fused_linear(*a, activation="silu", activation_dtype=kept), a, randn(40, 264, seed=6)
    yield lambda: fused_gated_mlp(*c, activation_dtype=kept), c, randn(40, 136, seed=7)


@pytest.mark.parametrize("kept", [None, FP8])
@pytest.mark.parametrize("unpack", [columns, spread, off])
def test_other_layouts(kept, unpack):
    for call, leaves, go in steps(kept):
        want = torch.autograd.grad(call(), leaves, go)
        # The weights stay as they are: their gradients take their layout.
        shapes = {tuple(t.shape) for t in leaves[1:]}
        with saved_tensors_hooks(lambda t: t, lambda t: t if tuple(t.shape) in shapes else unpack(t)):
            got = torch.autograd.grad(call(), leaves, go)
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("kept", [None, FP8])
@pytest.mark.parametrize("unpack", [lambda t: t[:-8], lambda t: t[:, :-8], lambda t: t.float(), lambda t: t.cpu(), lambda t: t[0]])
def test_other_tensors_are_refused(kept, unpack):
    """One saved tensor after the other is replaced; those of a residual's or bias's own are none."""
    for call, leaves, go in steps(kept):
        seen = []
        with saved_tensors_hooks(lambda t: t, lambda t: seen.append(t) or t):
            torch.autograd.grad(call(), leaves, go)
        for k, t in enumerate(seen):
            if unpack(t).dtype == t.dtype and unpack(t).shape == t.shape and unpack(t).device == t.device:
                continue  # fp32 scales as fp32
            count = iter(range(len(seen)))
            with saved_tensors_hooks(lambda t: t, lambda t: unpack(t) if next(count) == k else t):
                out = call()
                with pytest.raises((RuntimeError, ValueError), match="not what the forward saved|must be"):
                    torch.autograd.grad(out, leaves, go)
