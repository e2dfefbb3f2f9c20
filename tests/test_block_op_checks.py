"""What the operators torch.ops.mlpk.* of the block refuse when they are called by
themselves (fake tensors; no GPU needed) -- a kernel would read or write outside
the tensors."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlp_megakernel_b200  # noqa: F401  (registers the operators)

ops = torch.ops.mlpk
F16, F32, I32 = torch.float16, torch.float32, torch.int32


@pytest.fixture(autouse=True)
def fake():
    with FakeTensorMode():
        yield


def t(*shape, dtype=F16, device="cuda"):
    return torch.empty(*shape, dtype=dtype, device=device)


def refused(cases, kinds=(ValueError, TypeError, RuntimeError)):
    for k, call in enumerate(cases):
        with pytest.raises(kinds):
            call()
            pytest.fail(f"case {k} was not refused")


def test_norm():
    x, w = t(4, 8), t(8)
    assert [o.shape for o in ops.rms_norm(x, w, x, 1e-6)] == [(4, 8), (4,), (4, 8)]
    refused([lambda: ops.rms_norm(t(4, 0), None, None, 1e-6), lambda: ops.rms_norm(x, t(7), None, 1e-6),
             lambda: ops.rms_norm(x, w, t(3, 8), 1e-6), lambda: ops.rms_norm(x, w, None, -1.0),
             lambda: ops.rms_norm(t(4, 8, dtype=torch.float64), None, None, 1e-6),
             lambda: ops.rms_norm_fp8(x, w, None, 1e-6, 64), lambda: ops.rms_norm_fp8(x, w, None, 1e-6, -128)])


def test_norm_backward():
    x, w, rstd, g = t(4, 8), t(8), t(4, dtype=F32), t(4, 8)
    assert [o.shape for o in ops.rms_norm_bwd(x, None, w, rstd, g, None, True)] == [(4, 8), (8,)]
    refused([lambda: ops.rms_norm_bwd(x, None, w, t(3, dtype=F32), g, None, True),
             lambda: ops.rms_norm_bwd(x, None, w, t(4), g, None, True),
             lambda: ops.rms_norm_bwd(x, None, w, t(8, dtype=F32)[::2], g, None, True),
             lambda: ops.rms_norm_bwd(x, None, w, t(4, 1, dtype=F32), g, None, True),
             lambda: ops.rms_norm_bwd(x, None, w, rstd, t(3, 8), None, True),
             lambda: ops.rms_norm_bwd(x, None, w, rstd, t(4, 8, dtype=F32), None, True),
             lambda: ops.rms_norm_bwd(x, None, w, rstd, g, t(4, 7), True),
             lambda: ops.rms_norm_bwd(x, t(4, 8, dtype=F32), w, rstd, g, None, True),
             lambda: ops.rms_norm_bwd(x, None, t(9), rstd, g, None, True),
             lambda: ops.rms_norm_bwd(x, None, None, rstd, g, None, True)])


def test_sort():
    assert [o.shape for o in ops.expert_sort(t(4, 2, dtype=torch.int64), 3)] == [(4, 2), (4,)]
    refused([lambda: ops.expert_sort(t(4, 2, dtype=torch.int16), 3), lambda: ops.expert_sort(t(4, dtype=I32), 3),
             lambda: ops.expert_sort(t(4, 2, dtype=I32), 0), lambda: ops.expert_sort(t(4, 2, dtype=I32), 1025),
             lambda: ops.expert_sort(t(4, 0, dtype=I32), 3)])


PLANS = [lambda: (t(4, 2, dtype=torch.int64), t(4, dtype=I32)), lambda: (t(8, dtype=I32), t(4, dtype=I32)),
         lambda: (t(4, 2, dtype=I32), t(4, dtype=torch.int64)), lambda: (t(4, 2, dtype=I32), t(1, dtype=I32)),
         lambda: (t(4, 2, dtype=I32), t(2, 2, dtype=I32)), lambda: (t(4, 2, dtype=I32), t(8, dtype=I32)[::2]),
         lambda: (t(4, 2, dtype=I32, device="cpu"), t(4, dtype=I32)),
         lambda: (t(4, 2, dtype=I32), t(4, dtype=I32, device="cpu"))]


def test_rows():
    plan = t(4, 2, dtype=I32), t(4, dtype=I32)
    x, y, w, g = t(4, 8), t(8, 8), t(4, 2, dtype=F32), t(4, 8)
    assert ops.expert_dispatch(x, *plan).shape == (8, 8) and ops.expert_combine(y, w, *plan).shape == (4, 8)
    assert [o.shape for o in ops.expert_combine_bwd(g, y, w, *plan, True, True)] == [(8, 8), (4, 2)]
    refused([lambda: ops.expert_dispatch(t(3, 8), *plan), lambda: ops.expert_dispatch(t(4, 0), *plan),
             lambda: ops.expert_dispatch(t(32), *plan), lambda: ops.expert_dispatch(t(4, 8, dtype=torch.int8), *plan),
             lambda: ops.expert_combine(t(7, 8), w, *plan), lambda: ops.expert_combine(t(4, 8), None, *plan),
             lambda: ops.expert_combine(y, t(4, 3, dtype=F32), *plan),
             lambda: ops.expert_combine(y, t(4, 2, dtype=torch.bfloat16), *plan),
             lambda: ops.expert_combine_bwd(t(3, 8), y, w, *plan, True, True),
             lambda: ops.expert_combine_bwd(t(4, 9), y, w, *plan, True, True),
             lambda: ops.expert_combine_bwd(t(4, 8, dtype=F32), y, w, *plan, True, True),
             lambda: ops.expert_combine_bwd(g, t(7, 8), w, *plan, True, True),
             lambda: ops.expert_combine_bwd(g, y, t(8, dtype=F32), *plan, True, True),
             lambda: ops.expert_combine_bwd(g, y, None, *plan, True, True)])
    for bad in PLANS:
        plan = bad()
        refused([lambda: ops.expert_dispatch(x, *plan), lambda: ops.expert_combine(y, w, *plan),
                 lambda: ops.expert_combine_bwd(g, y, w, *plan, True, True)])
