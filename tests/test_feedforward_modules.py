"""The feed-forward modules with parameters of one type and inputs of another: the casts' shapes and types on fake tensors
here; values, and autocast, on the GPU in test_feedforward_modules_gpu.py."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlp_megakernel_b200 as m

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("params", [F16, BF16, F32])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_parameters_of_another_type(params, dtype):
    with FakeTensorMode():
        for module in (m.FusedLinear(16, 24), m.FusedLinear(16, 24, bias=False, activation="silu"), m.FusedGatedMLP(16, 32, 24)):
            for name, p in list(module.named_parameters()):
                setattr(module, name, torch.nn.Parameter(torch.empty(p.shape, dtype=params, device="cuda")))
            out = module(torch.empty(3, 16, dtype=dtype, device="cuda"), torch.empty(3, 24, dtype=F32, device="cuda"))
            assert out.dtype == dtype and out.shape == (3, 24) and out.requires_grad
