"""What the block operators refuse, and their shapes on fake tensors (CPU)."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlp_megakernel_b200 as m
from mlp_megakernel_b200 import _lib


@pytest.fixture
def fake():
    with FakeTensorMode() as mode:
        yield mode


def cuda(*shape, dtype=torch.float16, **more):
    return torch.empty(*shape, device="cuda", dtype=dtype, **more)


def test_cpu_tensors_raise():
    x = torch.zeros(4, 8)
    for call in (lambda: m.fused_rms_norm(x), lambda: m.fused_rms_norm_fp8(x),
                 lambda: m.expert_sort(torch.zeros(4, 2, dtype=torch.int64), 3),
                 lambda: m.FusedAdamW([torch.nn.Parameter(x)])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_norm_refusals(fake):
    x = cuda(4, 8)
    for bad, kind in ((lambda: m.fused_rms_norm(3.0), ValueError),
                      (lambda: m.fused_rms_norm(cuda(4, 8, dtype=torch.float64)), TypeError),
                      (lambda: m.fused_rms_norm(cuda(4, 0)), ValueError),
                      (lambda: m.fused_rms_norm(cuda(1, 32769)), ValueError),
                      (lambda: m.fused_rms_norm(x, cuda(7)), ValueError),
                      (lambda: m.fused_rms_norm(x, cuda(8, dtype=torch.bfloat16)), ValueError),
                      (lambda: m.fused_rms_norm(x, torch.empty(8, device="cpu", dtype=torch.float16)), ValueError),
                      (lambda: m.fused_rms_norm(x, residual=cuda(3, 8)), ValueError),
                      (lambda: m.fused_rms_norm(x, residual=cuda(4, 8, dtype=torch.float32)), ValueError),
                      (lambda: m.fused_rms_norm(x, eps=-1.0), ValueError),
                      (lambda: m.fused_rms_norm(x, eps=float("nan")), ValueError),
                      (lambda: m.fused_rms_norm_fp8(x, group=64), ValueError),
                      (lambda: m.fused_rms_norm_fp8(cuda(4, 8, requires_grad=True)), RuntimeError),
                      (lambda: m.FusedRMSNorm(0), ValueError)):
        with pytest.raises(kind):
            bad()


def test_expert_refusals(fake):
    ids = cuda(4, 2, dtype=torch.int64)
    plan = m.expert_sort(ids, 3)
    for bad, kind in ((lambda: m.expert_sort(cuda(4, dtype=torch.int64), 3), ValueError),
                      (lambda: m.expert_sort(cuda(4, 2, dtype=torch.int16), 3), TypeError),
                      (lambda: m.expert_sort(ids, 0), ValueError),
                      (lambda: m.expert_sort(ids, 1025), ValueError),
                      (lambda: m.expert_sort(cuda(4, 0, dtype=torch.int64), 3), ValueError),
                      (lambda: m.expert_dispatch(cuda(5, 8), plan), ValueError),
                      (lambda: m.expert_dispatch(cuda(4, 8, dtype=torch.float64), plan), TypeError),
                      (lambda: m.expert_dispatch(cuda(4, 8), m.ExpertPlan(ids, plan.offsets)), ValueError),
                      (lambda: m.expert_combine(cuda(4, 8), None, plan), ValueError),
                      (lambda: m.expert_combine(cuda(8, 8), cuda(4, 3), plan), ValueError),
                      (lambda: m.expert_combine(cuda(8, 8), cuda(4, 2, dtype=torch.bfloat16), plan), ValueError),
                      (lambda: m.FusedMLPExperts(num_experts=2, top=3), ValueError),
                      (lambda: m.FusedMLPExperts(capacity=0), ValueError)):
        with pytest.raises(kind):
            bad()


def test_adamw_refusals(fake):
    def param(*shape, **more):
        return torch.nn.Parameter(cuda(*shape, **more))

    p = param(8, 8)
    for bad, kind in ((lambda: m.FusedAdamW([p], state_bits=4), ValueError),
                      (lambda: m.FusedAdamW([p], lr=-1.0), ValueError),
                      (lambda: m.FusedAdamW([p], lr=torch.tensor(1.0, device="cpu")), ValueError),
                      (lambda: m.FusedAdamW([p], betas=(1.0, 0.9)), ValueError),
                      (lambda: m.FusedAdamW([p], betas=(0.9, -0.1)), ValueError),
                      (lambda: m.FusedAdamW([p], eps=-1e-8), ValueError),
                      (lambda: m.FusedAdamW([p], weight_decay=-0.1), ValueError),
                      (lambda: m.FusedAdamW([param(8, dtype=torch.float64)]), TypeError),
                      (lambda: m.FusedAdamW([torch.nn.Parameter(cuda(8, 9)[:, :8])]), ValueError)):
        with pytest.raises(kind):
            bad()


def test_a_refused_group_is_not_added(fake):
    opt = m.FusedAdamW([torch.nn.Parameter(cuda(8))])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(cuda(4))], "lr": -1.0})
    assert len(opt.param_groups) == 1


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_shapes_on_fake_tensors(fake, dtype):
    x, r = cuda(3, 5, 200, dtype=dtype), cuda(3, 5, 200, dtype=dtype)
    y, h = m.fused_rms_norm(x, cuda(200, dtype=dtype), residual=r)
    assert y.shape == h.shape == x.shape and y.dtype == h.dtype == dtype
    q, scale = m.fused_rms_norm_fp8(x, group=128)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (3, 5, 2)
    plan = m.expert_sort(cuda(7, 3, dtype=torch.int32), 5)
    assert plan.row_of.shape == (7, 3) and plan.offsets.shape == (6,) and plan.num_experts == 5
    xs = m.expert_dispatch(cuda(7, 40, dtype=dtype, requires_grad=True), plan)
    assert xs.shape == (21, 40) and xs.requires_grad
    out = m.expert_combine(xs, cuda(7, 3, dtype=torch.float32), plan)
    assert out.shape == (7, 40) and out.dtype == dtype


def test_c_calls_refuse_before_they_touch_the_device(built_lib):
    lib, a = built_lib, 256  # an aligned address that is never read
    sh, un, al, nu = (1, 2, 5, 6)
    for want, args in ((sh, (-1, 8, 0, a, None, None, 0, 1e-6, a, None, None, None)),
                       (sh, (4, 0, 0, a, None, None, 0, 1e-6, a, None, None, None)),
                       (un, (4, 32769, 0, a, None, None, 0, 1e-6, a, None, None, None)),
                       (un, (4, 8, 3, a, None, None, 0, 1e-6, a, None, None, None)),
                       (un, (4, 8, 0, a, None, a, 2, 1e-6, a, None, None, None)),
                       (nu, (4, 8, 0, None, None, None, 0, 1e-6, a, None, None, None)),
                       (nu, (4, 8, 0, a, a, None, 0, 1e-6, a, None, None, None)),
                       (al, (4, 8, 0, a + 2, None, None, 0, 1e-6, a, None, None, None)),
                       (0, (0, 8, 0, None, None, None, 0, 1e-6, None, None, None, None))):
        assert lib.mlpk_rms_norm(*args) == want
    assert lib.mlpk_rms_norm_fp8(4, 8, 0, a, None, None, 0, 1e-6, 64, a, a, None, None) == un
    assert lib.mlpk_rms_norm_fp8(4, 8, 0, a, None, None, 0, 1e-6, 0, a, None, None, None) == nu
    assert lib.mlpk_rms_norm_bwd(4, 8, 0, a, None, a, None, 0, a, None, a, a, a, 1 << 20, None) == nu  # no weight for dw
    assert lib.mlpk_rms_norm_bwd(4, 8, 0, a, None, a, a, 0, a, None, a, a, None, 0, None) == nu
    assert lib.mlpk_expert_sort(-1, 4, a, 8, a, a, None, 0, None) == sh
    assert lib.mlpk_expert_sort(8, 2000, a, 8, a, a, None, 0, None) == un
    assert lib.mlpk_expert_sort(8, 4, a, 2, a, a, None, 0, None) == un
    assert lib.mlpk_expert_sort(8, 4, a, 8, None, a, None, 0, None) == nu
    assert lib.mlpk_expert_sort(8, 4, a, 8, a + 4, a, None, 0, None) == al
    assert lib.mlpk_expert_dispatch(2 ** 30, 2, 8, 0, a, a, a, a, None) == sh
    assert lib.mlpk_expert_dispatch(4, 2, 8, 7, a, a, a, a, None) == un
    assert lib.mlpk_expert_dispatch(4, 2, 8, 0, a, a, None, a, None) == nu
    assert lib.mlpk_expert_combine(4, 2, 8, 0, a, a, 2, a, a, a, None) == un
    assert lib.mlpk_expert_combine(4, 2, 8, 0, a, None, 0, a, a, a + 8, None) == al
    assert lib.mlpk_expert_combine_bwd(4, 2, 8, 0, a, None, a, 0, a, a, a, a, None) == nu
    assert lib.mlpk_expert_combine_bwd(4, 2, 8, 0, a, a, a, 0, a, a, None, None, None) == 0  # nothing wanted
    one = (ctypes.c_int64 * 1)(300)
    off, bad_off, tick = (ctypes.c_int64 * 1)(0), (ctypes.c_int64 * 1)(100), (ctypes.c_int32 * 1)(0)
    ptr, none = _lib.ptr_array([a]), _lib.ptr_array([0])
    args = _lib.MlpkAdamwArgs(1e-3, 0.9, 0.999, 1e-8, 0.0, 0, None, None, None)
    state = _lib.MlpkAdamwState(32, a, a, None, None, None, a)
    b = ctypes.byref

    def step(count, numel, p, g, o, pd, gd, s):
        return lib.mlpk_adamw_step(count, numel, p, g, o, tick, pd, gd, b(s), b(args), None)

    assert step(-1, one, ptr, ptr, off, 0, 0, state) == sh
    assert step(1, one, ptr, ptr, off, 0, 2, state) == un
    assert step(1, one, ptr, ptr, off, 9, 9, state) in (un, 3, 4)
    assert step(1, one, ptr, none, off, 0, 0, state) == nu
    assert step(1, one, ptr, ptr, bad_off, 0, 0, state) == al
    assert step(1, one, ptr, ptr, off, 0, 0, _lib.MlpkAdamwState(16, a, a, None, None, None, a)) == un
    assert step(1, one, ptr, ptr, off, 0, 0, _lib.MlpkAdamwState(8, a, a, None, None, None, a)) == nu
    assert step(1, one, ptr, ptr, off, 1, 1, _lib.MlpkAdamwState(32, a, a, None, None, a, a)) == un
    assert step(0, None, None, None, None, 0, 0, state) == 0
