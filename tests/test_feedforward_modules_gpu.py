"""The feed-forward modules with parameters of another type than their input's or autocast's, forward and backward: the
bits of the calls with the parameters cast by hand, gradients in the parameters' types."""
import pytest
import torch

from mlp_megakernel_b200 import FusedGatedMLP, FusedLinear, fused_gated_mlp, fused_linear

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("params", [F16, BF16, F32])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("autocast", [False, True])
def test_parameters_of_another_type(params, dtype, autocast):
    torch.manual_seed(0)
    x = torch.randn(70, 72, device="cuda").to(dtype)
    for module in (FusedLinear(72, 40, activation="silu"), FusedLinear(72, 40, bias=False), FusedGatedMLP(72, 136, 40)):
        module = module.cuda().to(params)
        if getattr(module, "bias", None) is not None:
            torch.nn.init.normal_(module.bias)
        with torch.autocast("cuda", dtype=dtype, enabled=autocast):
            out = module(x.float() if autocast else x)
        go = torch.randn(70, 40, device="cuda").to(dtype)
        got = torch.autograd.grad(out, list(module.parameters()), go)
        leaves = {k: p.detach().to(dtype if k != "bias" or p.dtype != F32 else F32).requires_grad_() for k, p in module.named_parameters()}
        if isinstance(module, FusedLinear):
            want = fused_linear(x, leaves["weight"], leaves.get("bias"), activation=module.activation)
        else:
            want = fused_gated_mlp(x, leaves["w_gate"], leaves["w_up"], leaves["w_down"])
        wanted = torch.autograd.grad(want, list(leaves.values()), go)
        assert out.dtype == dtype and torch.equal(out, want)
        for g, w in zip(got, wanted):
            assert g.dtype == params and torch.equal(g, w.to(params))
