"""Values before the activation that the operands' type cannot hold: the forward has them in fp32, the backward as they
were kept, the nearest finite value.  Gradients are finite and those of the formula in 64 bits; tolerances as derived in
test_feedforward_gpu.py, with an activation's own error left out where its derivative is 0 or 1 beyond fp32's last place.

A linear layer's gradients are the formula's for z itself (every derivative is constant out there); a gate's are those of
the kept projections, which test_gated asks for, and exactly zero where the gate is shut.
"""
import pytest
import torch

from mlp_megakernel_b200 import _lib, feedforward as ff, fused_gated_mlp, fused_linear
from tests.test_feedforward_gpu import ACC, TINY, U, act64, close, kept64, make, product

pytestmark = pytest.mark.gpu
ops = torch.ops.mlpk
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
ACTS = [a for a in ff.ACTIVATIONS if a is not None]
ROWS = [5, 150, 700, 2000]  # the kernel for few rows, and tiles of 256


@pytest.fixture(autouse=True)
def status():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def linear(rows, act, keep, dtype, x, w, b, r, far):
    """A layer whose |z| is beyond `far` in some columns."""
    u = U[dtype]
    z, off = product(x.double(), w.double())
    if b is not None:
        z, off = z + b.double(), off + ACC * z.abs()
    out, *kept = ops.linear(x, w, b, r, ff.ACTIVATIONS[act], keep)
    v, s = (kept + [None])[:2]
    assert torch.isfinite(out).all() and torch.isfinite(kept64(v, s, z.shape[1])).all()
    outlier = z.abs() > far
    assert outlier.any(0).sum() >= 2
    if keep == 1:
        most = torch.finfo(dtype).max
        assert torch.equal(v[outlier].double(), most * z[outlier].sign()) and (v[~outlier].double().abs() < most).all()
    near = torch.where(outlier, z, kept64(v, s, z.shape[1]))  # the outliers as they are, not as they were kept
    _, slope, rel = act64(act, near)
    go = make(*z.shape, dtype=dtype, seed=5)
    dx, dw, db = ops.linear_bwd(go, x, None, w, v, s, ff.ACTIVATIONS[act], F32, True, True, True)
    dz = go.double() * slope
    room = torch.where(outlier, 0.0, rel * go.double().abs() * slope.abs().clamp(min=0.01)) + ACC * go.double().abs()
    close(db, dz.sum(0), room.sum(0) + (rows + 20) * ACC * dz.abs().sum(0), ACC, "db")
    room = room * (1 + u) + u * dz.abs() + TINY
    close(dx, *product(dz, w.double().t(), ea=room), u, "dx")
    close(dw, *product(x.double().t(), dz, eb=room), u, "dw")


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("keep", [1, 2])
def test_linear_beyond_fp16(rows, act, keep):
    x, w = make(rows, 72, dtype=F16, seed=1), make(72, 264, dtype=F16, seed=2, scale=0.1)
    x[:, 0] = 150
    w[0] = 0
    w[0, 3], w[0, 200] = 700, -700  # z near 105,000 and its negative
    r = make(rows, 264, dtype=F16, seed=4)
    if act != "sigmoid":
        r[:, 3] = -60000  # the output is finite in fp16
    linear(rows, act, keep, F16, x, w, None, r, 65520.0)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("act", [a for a in ACTS if a != "gelu_tanh"])
def test_linear_beyond_bf16(rows, act):
    x, w = make(rows, 72, dtype=BF16, seed=1), make(72, 264, dtype=BF16, seed=2, scale=0.1)
    b, r = make(264, dtype=F32, seed=3), make(rows, 264, dtype=BF16, seed=4)
    b[3], b[200] = 3.4e38, -3.4e38
    if act != "sigmoid":
        r[:, 3] = -3.3e38
    linear(rows, act, 1, BF16, x, w, b, r, 3.39618e38)


def gelu_far_out(rows, top, keep):
    x, w = make(rows, 72, dtype=BF16, seed=1), make(72, 264, dtype=BF16, seed=2, scale=0.1)
    b, r = make(264, dtype=F32, seed=3), make(rows, 264, dtype=BF16, seed=4)
    b[3], b[200] = top, -top
    n, z = 264, x.double() @ w.double() + b.double()
    out, *kept = ops.linear(x, w, b, r, ff.ACTIVATIONS["gelu_tanh"], keep)
    v, s = (kept + [None])[:2]
    go = make(rows, n, dtype=BF16, seed=5)
    dx, dw, db = ops.linear_bwd(go, x, None, w, v, s, ff.ACTIVATIONS["gelu_tanh"], F32, True, True, True)
    assert torch.isfinite(out).all() and all(torch.isfinite(t).all() for t in (dx, dw, db))
    far = z.abs() > 1e19
    assert far[:, 3].all() and far[:, 200].all() and not far[:, :3].any()
    near = torch.where(far, z, kept64(v, s, n))
    _, slope, rel = act64("gelu_tanh", near)
    assert (slope[:, 3] == 1).all() and (slope[:, 200] == 0).all()
    dz, u = go.double() * slope, U[BF16]
    room = torch.where(far, 0.0, rel * go.double().abs() * slope.abs().clamp(min=0.01)) + ACC * go.double().abs()
    close(db, dz.sum(0), room.sum(0) + (rows + 20) * ACC * dz.abs().sum(0), ACC, "db")
    room = room * (1 + u) + u * dz.abs() + TINY
    close(dx, *product(dz, w.double().t(), ea=room), u, "dx")
    close(dw, *product(x.double().t(), dz, eb=room), u, "dw")


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("top", [2e19, 1e22, 3e38])
@pytest.mark.parametrize("keep", [1, 2])
def test_gelu_where_the_square_overflows(rows, top, keep):
    """z^2 leaves fp32 above 1.8e19: the derivative is 1 or 0 there."""
    gelu_far_out(rows, top, keep)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("keep", [1, 2])
def test_gelu_next_to_the_largest_value(rows, keep):
    """3.38e38 in 8 bits is 256 x 2^120, beyond fp32: read back, it is fp32's largest value."""
    gelu_far_out(rows, 3.38e38, keep)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("act", [a for a in ACTS if a != "gelu_tanh"])
def test_linear_from_8_bits_next_to_the_largest_value(rows, act):
    x, w = make(rows, 72, dtype=BF16, seed=1), make(72, 264, dtype=BF16, seed=2, scale=0.1)
    b, r = make(264, dtype=F32, seed=3), make(rows, 264, dtype=BF16, seed=4)
    b[3], b[200] = 3.35e38, -3.35e38
    linear(rows, act, 2, BF16, x, w, b, r, 3.3e38)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_a_gate_from_8_bits_next_to_the_largest_value(rows, act):
    """A shut gate whose 8-bit value would be minus infinity in fp32."""
    x, wg, wu = make(rows, 72, dtype=BF16, seed=1), make(72, 264, dtype=BF16, seed=2, scale=0.1), make(72, 264, dtype=BF16, seed=3, scale=0.1)
    wd, go = make(264, 136, dtype=BF16, seed=4, scale=0.1), make(rows, 136, dtype=BF16, seed=5)
    x[:, 0], wg[0], wu[0] = 2.0 ** 64, 0, 0
    wg[0, 7] = -1.9765625 * 2.0 ** 63  # g is -3.36e38
    out, gk, sg, uk, su = ops.gated_mlp(x, wg, wu, wd, None, ff.ACTIVATIONS[act], 2)
    assert (kept64(gk, sg, 264)[:, 7] == -2.0 ** 128).all()
    got = ops.gated_mlp_bwd(go, None, None, wg, wu, wd, gk, sg, uk, su, ff.ACTIVATIONS[act], True, False, True)
    assert all(torch.isfinite(t).all() for t in (out, *got)) and not got[1][7].any()


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("keep", [1, 2])
def test_a_gelu_gate_where_the_square_overflows(rows, keep):
    """A gate of -1e22 is shut: no gradient of its column, and none that is not finite."""
    x, wg, wu = make(rows, 72, dtype=BF16, seed=1), make(72, 264, dtype=BF16, seed=2, scale=0.1), make(72, 264, dtype=BF16, seed=3, scale=0.1)
    wd, go = make(264, 136, dtype=BF16, seed=4, scale=0.1), make(rows, 136, dtype=BF16, seed=5)
    x[:, 0], wg[0] = 1e12, 0
    wg[0, 7] = -1e10
    wu[0] = 0
    out, *kept = ops.gated_mlp(x, wg, wu, wd, None, ff.ACTIVATIONS["gelu_tanh"], keep)
    gk, sg, uk, su = kept if keep == 2 else (kept[0], None, kept[1], None)
    dx, dwg, dwu, dwd = ops.gated_mlp_bwd(go, x, None, wg, wu, wd, gk, sg, uk, su, ff.ACTIVATIONS["gelu_tanh"], True, True, True)
    assert all(torch.isfinite(t).all() for t in (out, dx, dwg, dwu, dwd))
    assert not dwg[:, 7].any() and not dwu[:, 7].any() and not dwd[7].any()


def stored(ref, off, u):
    return off * (1 + u) + u * ref.abs() + TINY


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("keep", [1, 2])
def test_gated_beyond_fp16(rows, act, keep):
    """Columns of the hidden width: a gate far below and far above, a projection far above and below behind a shut gate."""
    u, k, h, n = U[F16], 72, 264, 136
    x = make(rows, k, dtype=F16, seed=1)
    x[:, 0], x[:, 1] = 30, 1
    wg, wu = (make(k, h, dtype=F16, seed=s, scale=0.1) for s in (2, 3))
    wd = make(h, n, dtype=F16, seed=4, scale=h ** -0.5)
    for w in (wg, wu):
        w[0] = 0
    shut, wide, over, under = 3, 70, 130, 200
    wg[0, shut], wg[0, wide] = -3500, 3500
    wu[:, wide] *= 2.0 ** -7  # h stays in fp16
    wu[0, over], wu[0, under] = 3500, -3500
    for c in (over, under):
        wg[:, c] = 0
        wg[1, c] = -18
    out, *kept = ops.gated_mlp(x, wg, wu, wd, None, ff.ACTIVATIONS[act], keep)
    gk, sg, uk, su = kept if keep == 2 else (kept[0], None, kept[1], None)
    assert all(torch.isfinite(t).all() for t in (out, kept64(gk, sg, h), kept64(uk, su, h)))
    go = make(rows, n, dtype=F16, seed=6, scale=2.0 ** -12)  # no gradient leaves fp16
    got = ops.gated_mlp_bwd(go, x, None, wg, wu, wd, gk, sg, uk, su, ff.ACTIVATIONS[act], True, True, True)
    assert all(torch.isfinite(t).all() for t in got)
    dx, dwg, dwu, dwd = got
    if keep == 1:
        for t, c, sign in ((gk, shut, -1), (gk, wide, 1), (uk, over, 1), (uk, under, -1)):
            assert (t[:, c] == sign * 65504.0).all()
    assert not dwg[:, shut].any() and not dwu[:, shut].any() and not dwd[shut].any()
    g, up = kept64(gk, sg, h), kept64(uk, su, h)
    a, slope, rel = act64(act, g)
    rel = torch.where(g.abs() > 1e4, ACC, rel)
    dh, ed = product(go.double(), wd.double().t())
    h64, du, dg = a * up, dh * a, dh * up * slope
    eh = stored(h64, (rel * a.abs() + ACC) * up.abs() + ACC * h64.abs(), u)
    eu = stored(du, ed * a.abs() + dh.abs() * (rel * a.abs() + ACC) + ACC * du.abs(), u)
    slope_off = rel * slope.abs().clamp(min=0.01) + ACC
    eg = stored(dg, (ed * slope.abs() + (ed + dh.abs()) * slope_off) * up.abs() + 2 * ACC * dg.abs(), u)
    close(dwd, *product(h64.t(), go.double(), ea=eh.t()), u, "dw_down")
    close(dwg, *product(x.double().t(), dg, eb=eg), u, "dw_gate")
    close(dwu, *product(x.double().t(), du, eb=eu), u, "dw_up")
    (r1, o1), (r2, o2) = product(dg, wg.double().t(), ea=eg), product(du, wu.double().t(), ea=eu)
    size = dg.abs() @ wg.double().abs().t() + du.abs() @ wu.double().abs().t()
    close(dx, r1 + r2, o1 + o2 + h * ACC * size, u, "dx")


@pytest.mark.parametrize("rows", ROWS)
def test_hidden_values_next_to_the_largest(rows):
    """h is 65,491 from the fp32 projections, 65,536 from the kept ones (256.25 x 255.75): formed again, it is 65,504."""
    x, wd = torch.zeros(rows, 16, device="cuda", dtype=F16), torch.full((8, 8), 2.0 ** -10, device="cuda", dtype=F16)
    x[:, :2] = 1
    wg, wu = torch.zeros(16, 8, device="cuda", dtype=F16), torch.zeros(16, 8, device="cuda", dtype=F16)
    wg[0], wg[1], wu[0], wu[1] = 256, 0.126, 255.5, 0.2
    wd.requires_grad_()
    out = fused_gated_mlp(x, wg, wu, wd, activation=None)
    assert torch.isfinite(out).all()
    go = torch.full_like(out, 2.0 ** -12)
    dwd, = torch.autograd.grad(out, wd, go)
    assert torch.equal(dwd, torch.full_like(dwd, 65504 * rows * 2.0 ** -12))


def test_infinities_and_nan_are_kept():
    for rows in ROWS:
        for dtype in (F16, BF16):
            x, w = make(rows, 72, dtype=dtype, seed=1), make(72, 136, dtype=dtype, seed=2, scale=0.1)
            w[:, 5] = w[:, 5].abs()
            x[2], x[3, 4] = float("nan"), float("inf")
            _, z = ops.linear(x, w, None, None, 2, 1)
            _, g, u = ops.gated_mlp(x, w, w, w.t().contiguous(), None, 2, 1)
            for t in (z, g, u):
                assert t[2].isnan().all() and t[3, 5] == float("inf") and not torch.isfinite(t[3]).any()


def test_the_public_calls():
    """The layer and the block through autograd, fp16, with outliers: no gradient that is not finite."""
    x, w = make(90, 72, dtype=F16, seed=1), make(72, 136, dtype=F16, seed=2, scale=0.1)
    x[:, 0], w[0] = 300, 0
    w[0, 7] = -350
    wd = make(136, 72, dtype=F16, seed=3, scale=0.1)
    for f in (lambda a, b: fused_linear(a, b, activation="silu"), lambda a, b: fused_linear(a, b, activation="gelu_tanh"),
              lambda a, b: fused_gated_mlp(a, b, b, wd), lambda a, b: fused_gated_mlp(a, b, b, wd, activation="gelu_tanh")):
        a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
        out = f(a, b)
        got = torch.autograd.grad(out, (a, b), torch.ones_like(out))
        assert torch.isfinite(out).all() and all(torch.isfinite(t).all() for t in got)
