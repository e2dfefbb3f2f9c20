"""What the feed-forward operators refuse, and their shapes on fake tensors (CPU)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlp_megakernel_b200 as m
from mlp_megakernel_b200 import _lib

ops = torch.ops.mlpk
BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.fixture
def fake():
    with FakeTensorMode() as mode:
        yield mode


def t(*shape, dtype=F16, device="cuda", **more):
    return torch.empty(*shape, dtype=dtype, device=device, **more)


def refused(cases):
    for k, (call, kind) in enumerate(cases):
        with pytest.raises(kind):
            call()
            pytest.fail(f"case {k} was not refused")


def test_cpu_tensors_raise():
    x, w = torch.zeros(4, 8, dtype=F16), torch.zeros(8, 8, dtype=F16)
    for call in (lambda: m.fused_linear(x, w), lambda: m.fused_gated_mlp(x, w, w, w), lambda: m.fp8_checkpoint(x),
                 lambda: m.fp8_restore(x.to(FP8), torch.ones(4, 1)), lambda: m.FusedLinear(8, 8)(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_linear_refusals(fake):
    x, w = t(4, 16), t(16, 24)
    refused([(lambda: m.fused_linear(3.0, w), ValueError), (lambda: m.fused_linear(t(4, 16, dtype=F32), w), TypeError),
             (lambda: m.fused_linear(t(4, 12), t(12, 24)), ValueError),      # 12 is not a multiple of 8
             (lambda: m.fused_linear(t(4, 0), t(0, 24)), ValueError), (lambda: m.fused_linear(x, t(16, 20)), ValueError),
             (lambda: m.fused_linear(x, t(24, 24)), ValueError), (lambda: m.fused_linear(x, t(16)), ValueError),
             (lambda: m.fused_linear(x, t(16, 24, dtype=BF16)), ValueError),
             (lambda: m.fused_linear(x, t(16, 24, device="cpu")), ValueError),
             (lambda: m.fused_linear(x, w, t(16)), ValueError), (lambda: m.fused_linear(x, w, t(24, dtype=BF16)), ValueError),
             (lambda: m.fused_linear(x, w, residual=t(4, 16)), ValueError),
             (lambda: m.fused_linear(x, w, residual=t(4, 24, dtype=F32)), ValueError),
             (lambda: m.fused_linear(x, w, activation="gelu"), ValueError),
             (lambda: m.fused_linear(x, w, activation_dtype=F32), TypeError),
             (lambda: m.fused_linear(x, w, activation_dtype=torch.float8_e5m2), TypeError),
             (lambda: m.FusedLinear(12, 8), ValueError), (lambda: m.FusedLinear(8, 8, activation="tanh"), ValueError),
             (lambda: m.FusedLinear(8, 8, activation_dtype=F16), TypeError)])


def test_gated_refusals(fake):
    x, g, d = t(4, 16), t(16, 24), t(24, 16)
    refused([(lambda: m.fused_gated_mlp(x, g, t(16, 32), d), ValueError), (lambda: m.fused_gated_mlp(x, g, g, t(16, 16)), ValueError),
             (lambda: m.fused_gated_mlp(x, g, g, t(24, 12)), ValueError),
             (lambda: m.fused_gated_mlp(x, g, t(16, 24, dtype=BF16), d), ValueError),
             (lambda: m.fused_gated_mlp(t(4, 16, dtype=F32), g, g, d), TypeError),
             (lambda: m.fused_gated_mlp(x, g, g, d, residual=t(4, 24)), ValueError),
             (lambda: m.fused_gated_mlp(x, g, g, d, activation="swish"), ValueError),
             (lambda: m.FusedGatedMLP(16, 20), ValueError), (lambda: m.FusedGatedMLP(16, 24, out_features=4), ValueError)])


def test_checkpoint_refusals(fake):
    q, s = t(4, 200, dtype=FP8), t(4, 2, dtype=F32)
    refused([(lambda: m.fp8_checkpoint(t(4, 8, dtype=torch.float64)), TypeError), (lambda: m.fp8_checkpoint(t(4, 0)), ValueError),
             (lambda: m.fp8_checkpoint(t(4, 8, requires_grad=True)), RuntimeError),
             (lambda: m.fp8_restore(t(4, 200), s), ValueError), (lambda: m.fp8_restore(q, t(4, 1, dtype=F32)), ValueError),
             (lambda: m.fp8_restore(q, t(4, 2)), ValueError), (lambda: m.fp8_restore(q, s, torch.float64), TypeError)])


def test_operators_check_their_tensors(fake):
    x, w, go, kept = t(4, 16), t(16, 24), t(4, 24), t(4, 24)
    wide, scale = t(4, 128, dtype=FP8), t(4, 1, dtype=F32)
    ok = lambda: ops.linear_bwd(go, x, None, w, kept, None, 2, F16, True, True, True)  # noqa: E731
    assert [o.shape for o in ok()] == [(4, 16), (16, 24), (24,)]
    assert [o.shape for o in ops.linear_bwd(go, None, None, w, wide, scale, 2, F32, True, False, True)] == [(4, 16), (24,)]
    kinds = (ValueError, TypeError, RuntimeError)

    def bwd(go=go, x=x, xs=None, w=w, z=kept, zs=None, act=2, db=F16, want=(True, True, True)):
        return lambda: ops.linear_bwd(go, x, xs, w, z, zs, act, db, *want)

    refused([(f, kinds) for f in (bwd(z=None), bwd(z=t(4, 16)), bwd(z=t(3, 24)), bwd(z=wide), bwd(z=wide, zs=t(4, 2, dtype=F32)),
                                  bwd(z=t(4, 24, dtype=FP8), zs=scale), bwd(z=kept, zs=scale), bwd(z=t(4, 24, dtype=BF16)),
                                  bwd(z=t(4, 48)[:, ::2]), bwd(x=None), bwd(x=t(5, 16)), bwd(x=t(4, 24)), bwd(x=t(4, 16, dtype=BF16)),
                                  bwd(x=t(4, 16, dtype=FP8)), bwd(x=t(4, 16, dtype=FP8), xs=t(4, 2, dtype=F32)), bwd(w=t(16, 16)),
                                  bwd(act=6), bwd(act=-1), bwd(db=BF16), bwd(go=t(4, 24, dtype=F32)))]
            + [(lambda: ops.linear(x, w, None, None, 7, 0), kinds), (lambda: ops.linear(x, w, None, None, 2, 3), kinds)])
    g, d = t(16, 24), t(24, 16)
    gk, go = t(4, 24), t(4, 16)

    def gated(go=go, x=x, xs=None, g=g, u=g, d=d, gk=gk, gs=None, uk=gk, us=None, act=2, want=(True, True, True)):
        return lambda: ops.gated_mlp_bwd(go, x, xs, g, u, d, gk, gs, uk, us, act, *want)

    assert [o.shape for o in gated()()] == [(4, 16), (16, 24), (16, 24), (24, 16)]
    refused([(f, kinds) for f in (gated(go=t(4, 24)), gated(g=t(16, 16)), gated(u=t(16, 32)), gated(d=t(32, 16)), gated(gk=t(4, 16)),
                                  gated(uk=t(5, 24)), gated(gk=wide, gs=scale), gated(gk=wide, uk=wide), gated(x=None),
                                  gated(x=t(4, 24)), gated(x=t(3, 16)), gated(act=9), gated(uk=t(24, 4).t()))])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_shapes_on_fake_tensors(fake, dtype):
    x, w = t(3, 5, 64, dtype=dtype, requires_grad=True), t(200, 64, dtype=dtype, requires_grad=True)
    out = m.fused_linear(x, w.t(), t(200, dtype=F32), activation="silu", residual=t(3, 5, 200, dtype=dtype))
    assert out.shape == (3, 5, 200) and out.dtype == dtype and out.requires_grad
    x, w = x.detach(), w.detach()
    dx, dw = ops.linear_bwd(out.detach(), x, None, w.t(), t(15, 200, dtype=dtype), None, 2, dtype, True, True, False)
    assert dx.shape == x.shape and dw.shape == (64, 200) and dw.stride() == w.t().stride()
    up, down = t(64, 72, dtype=dtype, requires_grad=True), t(72, 40, dtype=dtype)
    for kept in (None, FP8):
        out = m.fused_gated_mlp(x, up, up, down, activation_dtype=kept)
        assert out.shape == (3, 5, 40) and out.requires_grad
    q, scale = m.fp8_checkpoint(t(3, 5, 300, dtype=dtype))
    assert q.dtype == FP8 and q.shape == (3, 5, 300) and scale.shape == (3, 5, 3)
    assert m.fp8_restore(q, scale, F32).shape == (3, 5, 300)


def test_c_calls_refuse_before_they_touch_the_device(built_lib):
    lib, a = built_lib, 256  # an aligned address that is never read
    sh, un, al, nu = 1, 2, 5, 6
    one, two, none, odd = (_lib.ptr_array(p) for p in ([a], [a, a], [0], [a + 2]))

    def linear(rows=4, k=16, n=24, dt=2, x=a, w=a, layout=0, b=None, bdt=2, act=0, r=None, out=a, keep=0, z=None, zs=None):
        return lib.mlpk_linear(rows, k, n, dt, x, w, layout, b, bdt, act, r, out, keep, z, zs, None, 0, None)

    for want, more in ((sh, dict(rows=-1)), (sh, dict(rows=2 ** 31)), (sh, dict(k=0)), (un, dict(k=12)), (un, dict(n=20)),
                       (un, dict(dt=1)), (un, dict(layout=2)), (un, dict(act=6)), (un, dict(act=-1)), (un, dict(keep=3)),
                       (un, dict(b=a, bdt=0)), (nu, dict(x=None)), (nu, dict(out=None)), (nu, dict(keep=1)),
                       (nu, dict(keep=2, z=a)), (al, dict(w=a + 8)), (al, dict(r=a + 2)), (al, dict(b=a + 4, bdt=1)),
                       (0, dict(rows=0, x=None, w=None, out=None))):
        assert linear(**more) == want, more
    assert lib.mlpk_linear_dz(4, 20, 2, 2, a, 1, a, None, a, None, 2, None, 0, None) == un
    assert lib.mlpk_linear_dz(4, 24, 2, 2, a, 0, None, None, a, None, 2, None, 0, None) == nu
    assert lib.mlpk_linear_dz(4, 24, 2, 2, a, 2, a, None, a, None, 2, None, 0, None) == nu
    assert lib.mlpk_linear_dz(4, 24, 2, 0, a, 0, None, None, None, a, 2, None, 0, None) == nu  # no workspace for db
    assert lib.mlpk_linear_dz(4, 24, 2, 0, a, 0, None, None, None, None, 2, None, 0, None) == 0  # nothing wanted
    assert lib.mlpk_linear_dx(4, 16, 24, 2, 3, two, two, 0, a, None, 0, None) == sh
    assert lib.mlpk_linear_dx(4, 16, 24, 2, 1, none, one, 0, a, None, 0, None) == nu
    assert lib.mlpk_linear_dx(4, 16, 24, 2, 1, odd, one, 0, a, None, 0, None) == al
    assert lib.mlpk_linear_dx(4, 16, 24, 2, 1, None, one, 0, a, None, 0, None) == nu
    assert lib.mlpk_linear_dx(0, 16, 24, 2, 1, none, one, 0, None, None, 0, None) == 0
    assert lib.mlpk_linear_dw(4, 16, 24, 2, 0, a, one, one, 0, None, 0, None) == sh
    assert lib.mlpk_linear_dw(4, 16, 24, 2, 1, None, one, one, 0, None, 0, None) == nu
    assert lib.mlpk_linear_dw(0, 16, 24, 2, 1, None, none, none, 0, None, 0, None) == nu
    assert lib.mlpk_linear_dw_workspace_size(-1, 16, 24, 2, 1, 0) == -1
    assert lib.mlpk_linear_dx_workspace_size(4, 16, 24, 2, 1, 5) == -1
    assert lib.mlpk_gated(4, 16, 24, 2, 2, a, a, None, 0, a, 0, None, None, None, None, None) == nu
    assert lib.mlpk_gated(4, 16, 24, 2, 2, a, a, a, 0, a, 1, a, None, None, None, None) == nu
    assert lib.mlpk_gated(4, 16, 24, 2, 2, a, a, a, 0, a, 2, a, a, a, None, None) == nu
    assert lib.mlpk_gated_bwd(4, 24, 16, 2, 2, a, a, 0, 0, a, None, a, None, a, a, a, None) == un  # nothing was kept
    assert lib.mlpk_gated_bwd(4, 24, 16, 2, 2, a, a, 0, 2, a, a, a, None, a, a, a, None) == nu
    assert lib.mlpk_gated_bwd(4, 24, 16, 2, 2, a, a, 0, 1, a, None, a, None, a, a, a + 8, None) == al
    assert lib.mlpk_fp8_checkpoint(4, 0, 2, a, a, a, None) == sh and lib.mlpk_fp8_checkpoint(4, 8, 5, a, a, a, None) == un
    assert lib.mlpk_fp8_checkpoint(4, 8, 1, a, None, a, None) == nu and lib.mlpk_fp8_checkpoint(4, 8, 1, a, a, a + 4, None) == al
    assert lib.mlpk_fp8_restore(-1, 8, 1, a, a, a, None) == sh and lib.mlpk_fp8_restore(4, 8, 1, a, a, None, None) == nu
    assert [lib.mlpk_fp8_pitch(w) for w in (0, 1, 128, 129)] == [-1, 128, 128, 256]
