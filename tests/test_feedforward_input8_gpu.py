"""The weights' gradients from an input kept in 8 bits: x^T dz with the values that the 8-bit numbers stand for, against
the formula in 64 bits (tolerances as derived in test_feedforward_gpu.py; restored to fp16, a value below its normal range
is off by 2^-25, in bf16 by nothing)."""
import pytest
import torch

from mlp_megakernel_b200 import feedforward as ff, fp8_checkpoint
from tests.test_feedforward_gpu import ACC, TINY, U, act64, close, kept64, layout, make, product, status  # noqa: F401

pytestmark = pytest.mark.gpu
ops = torch.ops.mlpk
SHAPES = [(1, 8, 8), (37, 72, 40), (150, 200, 264), (700, 328, 776), (2000, 136, 2056), (3000, 1288, 520)]


def step_off(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 0.0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("transposed", [False, True])
def test_linear(shape, dtype, transposed):
    rows, k, n = shape
    u, act = U[dtype], "silu"
    x = make(rows, k, dtype=dtype, seed=1) * torch.logspace(-3, 1, k, device="cuda").to(dtype)
    w, go = layout(make(k, n, dtype=dtype, seed=2, scale=k ** -0.5), transposed), make(rows, n, dtype=dtype, seed=3)
    _, z = ops.linear(x, w, None, None, ff.ACTIVATIONS[act], 1)
    q, scale = fp8_checkpoint(x)
    dw, = ops.linear_bwd(go, q, scale, w, z, None, ff.ACTIVATIONS[act], dtype, False, True, False)
    _, slope, rel = act64(act, z.double())
    dz = go.double() * slope
    room = rel * go.double().abs() * slope.abs().clamp(min=0.01) + ACC * go.double().abs()
    room = room * (1 + u) + u * dz.abs() + TINY
    kept = kept64(q, scale, k)
    close(dw, *product(kept.t(), dz, ea=torch.full_like(kept.t(), step_off(dtype)), eb=room), u, "dw")


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", list(U))
def test_gated(shape, dtype):
    rows, k, h = shape
    u, act, n = U[dtype], "gelu_tanh", 40
    x = make(rows, k, dtype=dtype, seed=1) * torch.logspace(-3, 1, k, device="cuda").to(dtype)
    wg, wu, wd = (make(*s, dtype=dtype, seed=2 + i, scale=s[0] ** -0.5) for i, s in enumerate(((k, h), (k, h), (h, n))))
    go = make(rows, n, dtype=dtype, seed=5)
    _, gk, uk = ops.gated_mlp(x, wg, wu, wd, None, ff.ACTIVATIONS[act], 1)
    q, scale = fp8_checkpoint(x)
    dwg, dwu = ops.gated_mlp_bwd(go, q, scale, wg, wu, wd, gk, None, uk, None, ff.ACTIVATIONS[act], False, True, False)
    g, up = gk.double(), uk.double()
    a, slope, rel = act64(act, g)
    dh, ed = product(go.double(), wd.double().t())
    du, dg = dh * a, dh * up * slope
    stored = lambda ref, off: off * (1 + u) + u * ref.abs() + TINY  # noqa: E731
    eu = stored(du, ed * a.abs() + dh.abs() * (rel * a.abs() + ACC) + ACC * du.abs())
    slope_off = rel * slope.abs().clamp(min=0.01) + ACC
    eg = stored(dg, (ed * slope.abs() + (ed + dh.abs()) * slope_off) * up.abs() + 2 * ACC * dg.abs())
    kept = kept64(q, scale, k)
    off = torch.full_like(kept.t(), step_off(dtype))
    close(dwg, *product(kept.t(), dg, ea=off, eb=eg), u, "dw_gate")
    close(dwu, *product(kept.t(), du, ea=off, eb=eu), u, "dw_up")
