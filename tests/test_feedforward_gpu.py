"""The feed-forward products against the formulas in 64 bits.

Tolerances.  u is the unit roundoff of the operands' type (2^-11 fp16, 2^-8
bf16).  A product of K terms is summed in fp32, each addition off by one unit of
its last place at most (tensor cores truncate): |error| <= (K + 2) 2^-23 sum|a b|
=: acc.  The activations have slopes of 1.13 at most, their derivatives slopes of
0.8; both are off by 8 2^-23 (1 + |z|^3) of themselves (the exponent's argument)
or, softplus, by 6e-5 (its polynomial), and by 2^-22 absolutely.  Every rounding
of a stored value adds u of it, and 2^-25 (half of fp16's smallest step).  What a
forward keeps is checked against z; the backward's reference starts from the
values that were kept, so that no tolerance has to pass through their rounding.
"""
import math

import pytest
import torch

from mlp_megakernel_b200 import _lib, feedforward as ff, fp8_checkpoint, fp8_restore, fused_gated_mlp, fused_linear

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ACC, TINY = 2.0 ** -23, 2.0 ** -25
ops = torch.ops.mlpk
FP8 = torch.float8_e4m3fn
ACTS = list(ff.ACTIVATIONS)


@pytest.fixture(autouse=True)
def status():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def make(*shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


def act64(kind, z):
    """(activation, derivative, what each may be off by beside the argument's error)."""
    if kind is None:
        return z, torch.ones_like(z), torch.zeros_like(z)
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double(), torch.zeros_like(z)
    off = 8 * ACC * (1 + z.abs().clamp(max=100) ** 3)
    if kind == "softplus":
        s = torch.sigmoid(z)
        return torch.nn.functional.softplus(z, threshold=1000.0), s, off + 6e-5
    if kind == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        d = 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
        return 0.5 * z * (1 + t), d, off
    s = torch.sigmoid(z)
    return (s, s * (1 - s), off) if kind == "sigmoid" else (z * s, s + z * s * (1 - s), off)


def product(a, b, ea=None, eb=None):
    """(a b, how far the kernel's may be off) for operands that are off by ea, eb."""
    ref, size = a @ b, a.abs() @ b.abs()
    off = (a.shape[1] + 2) * ACC * size
    if ea is not None:
        off = off + ea @ b.abs()
    if eb is not None:
        off = off + a.abs() @ eb
    return ref, off


def close(got, ref, off, u, what=""):
    room = off * (1 + u) + u * ref.abs() + TINY
    over = ((got.double() - ref).abs() - room).max().item() if ref.numel() else 0.0
    assert over <= 0, f"{what} is off by {over} more than allowed"


def kept64(v, scale, width):
    if scale is None:
        return v.double()
    return v.double()[:, :width] * scale.double().repeat_interleave(128, dim=1)[:, :width]


def check_kept(v, scale, ref, off, u):
    """Within half a step of its type; 8 bits: 1/16 of the value or 2^-10 of the scale, and the scale as defined."""
    rows, width = ref.shape
    got = kept64(v, scale, width)
    if scale is None:
        return close(v, ref, off, u, "kept")
    each = scale.double().repeat_interleave(128, dim=1)[:, :width]
    over = ((got - ref).abs() - off * 1.07 - 2.0 ** -4 * ref.abs() - 2.0 ** -10 * each).max().item()
    assert over <= 0, f"kept is off by {over} more than allowed"
    groups = -(-width // 128)
    pad = torch.nn.functional.pad
    most, room = (pad(t, (0, groups * 128 - width)).view(rows, groups, 128).amax(-1) for t in (ref.abs(), off))
    assert torch.equal(torch.frexp(scale)[0], torch.full_like(scale, 0.5))  # a power of two
    s = scale.double()
    assert ((most - room) / s <= 448).all() and ((most + room) / s > 224).all()


def layout(w, transposed):
    return w.t().contiguous().t() if transposed else w


def linear_case(rows, k, n, dtype, act, bias, residual, transposed=False, keep=0, scale=1.0):
    x, w = make(rows, k, dtype=dtype, seed=1, scale=scale), layout(make(k, n, dtype=dtype, seed=2, scale=k ** -0.5), transposed)
    b = None if bias is None else make(n, dtype=bias, seed=3)
    r = make(rows, n, dtype=dtype, seed=4) if residual else None
    z, off = product(x.double(), w.double())
    if b is not None:
        z, off = z + b.double(), off + ACC * z.abs()
    out, *kept = ops.linear(x, w, b, r, ff.ACTIVATIONS[act], keep)
    a, _, rel = act64(act, z)
    ref, room = a, 1.13 * off + rel * a.abs() + ACC
    if r is not None:
        ref, room = ref + r.double(), room + ACC * (ref.abs() + r.double().abs())
    close(out, ref, room, U[dtype], "out")
    v, s = (kept + [None, None])[:2]
    if keep:
        check_kept(v, s, z, off, U[dtype])
    go = make(rows, n, dtype=dtype, seed=5)
    dx, dw, db = ops.linear_bwd(go, x, None, w, v, s, ff.ACTIVATIONS[act], bias or dtype, True, True, True) if keep or act is None \
        else (None, None, None)
    if dx is None:
        return
    dz, room = go.double(), torch.zeros_like(z)
    if act is not None:
        _, slope, rel = act64(act, kept64(v, s, n))
        dz = dz * slope
        room = rel * go.double().abs() * slope.abs().clamp(min=0.01) + ACC * go.double().abs()
    ref = dz.sum(0)
    close(db, ref, room.sum(0) + (rows + 20) * ACC * dz.abs().sum(0), U.get(db.dtype, ACC), "db")
    if act is not None:
        room = room * (1 + U[dtype]) + U[dtype] * dz.abs() + TINY  # dz as stored
    close(dx, *product(dz, w.double().t(), ea=room), U[dtype], "dx")
    close(dw, *product(x.double().t(), dz, eb=room), U[dtype], "dw")
    assert dw.stride() == w.stride()


SHAPES = [(1, 8, 8), (1, 64, 256), (3, 72, 40), (17, 128, 136), (64, 256, 256), (127, 200, 1000), (129, 1000, 264),
          (256, 64, 512), (257, 520, 248), (300, 4096, 128), (1000, 328, 776), (2000, 136, 2056)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", list(U))
def test_linear(shape, dtype):
    linear_case(*shape, dtype, None, None, False)
    linear_case(*shape, dtype, "silu", dtype, True, keep=1)
    linear_case(*shape, dtype, "gelu_tanh", torch.float32, False, keep=2, transposed=True)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("keep", [1, 2])
@pytest.mark.parametrize("dtype", list(U))
def test_linear_activations(act, keep, dtype):
    linear_case(333, 192, 456, dtype, act, dtype, True, keep=keep if act else 0, scale=3.0)


@pytest.mark.parametrize("shape", [(300, 4096, 128), (257, 2056, 136), (520, 4096, 128), (513, 2056, 136), (1000, 4096, 1032),
                                   (700, 5000, 264), (2100, 4096, 136), (2305, 5000, 264), (4000, 4096, 520)])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", list(U))
def test_linear_whose_last_tiles_are_shared_out(shape, act, dtype):
    """Long reductions of few tiles: shares of a tile meet in a second kernel, which runs the epilogue."""
    if shape in ((2100, 4096, 136), (2305, 5000, 264)):  # others may go elsewhere, or end earlier whole
        assert _lib.lib().mlpk_linear_workspace_size(*shape, 0 if dtype == torch.float16 else 2, 0, 0) > 0
    linear_case(*shape, dtype, act, dtype, True)
    linear_case(*shape, dtype, act, torch.float32, False, transposed=True)


@pytest.mark.parametrize("shape", [(513, 136, 3088), (513, 136, 3872), (600, 200, 4600), (769, 520, 4656), (2000, 264, 1288),
                                   (2500, 72, 1400), (520, 2000, 1288), (20000, 264, 136)])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dtype", list(U))
def test_tiles_of_any_width(shape, transposed, dtype):
    """One turn of tiles of 160, 192 and 224 columns, the last one cut off by the edge."""
    linear_case(*shape, dtype, None, None, False, transposed=transposed)
    linear_case(*shape, dtype, "gelu_tanh", dtype, True, keep=1, transposed=transposed)


@pytest.mark.parametrize("shape", [(129, 2056, 520), (145, 4096, 264), (208, 1032, 1000), (257, 4096, 136), (300, 2048, 1000),
                                   (400, 4104, 264), (512, 4096, 136), (1000, 4096, 1000), (1999, 4096, 520)])
@pytest.mark.parametrize("dtype", list(U))
def test_long_reductions_of_some_hundred_rows(shape, dtype):
    """Rows that fill one tile or several of the kernel for few rows, the last one partly."""
    rows, k, n = shape
    linear_case(rows, k, n, dtype, None, None, False)
    linear_case(rows, k, n, dtype, "gelu_tanh", dtype, True, keep=1)
    linear_case(rows, k, n, dtype, "silu", torch.float32, False, keep=2, transposed=True)
    gated_case(rows, k, n, 136, dtype, "silu", True, 0)
    gated_case(rows, k, n, 136, dtype, "gelu_tanh", False, 1, transposed=(True, False, True))


def gated_case(rows, k, h, n, dtype, act, residual, keep, transposed=(False, False, False)):
    u = U[dtype]
    x = make(rows, k, dtype=dtype, seed=1)
    wg, wu = (layout(make(k, h, dtype=dtype, seed=s, scale=k ** -0.5), t) for s, t in ((2, transposed[0]), (3, transposed[1])))
    wd = layout(make(h, n, dtype=dtype, seed=4, scale=h ** -0.5), transposed[2])
    r = make(rows, n, dtype=dtype, seed=5) if residual else None
    out, *kept = ops.gated_mlp(x, wg, wu, wd, r, ff.ACTIVATIONS[act], keep)
    (g, eg), (up, eu) = product(x.double(), wg.double()), product(x.double(), wu.double())
    a, _, rel = act64(act, g)
    ea = 1.13 * eg + rel * a.abs() + ACC
    h64 = a * up
    eh = ea * up.abs() + a.abs() * eu + ACC * h64.abs()
    ref, room = product(h64, wd.double(), ea=eh * (1 + u) + u * h64.abs() + TINY)
    if r is not None:
        ref, room = ref + r.double(), room + ACC * (ref.abs() + r.double().abs())
    close(out, ref, room, u, "out")
    if not keep:
        return
    gk, sg, uk, su = kept if keep == 2 else (kept[0], None, kept[1], None)
    check_kept(gk, sg, g, eg, u)
    check_kept(uk, su, up, eu, u)
    go = make(rows, n, dtype=dtype, seed=6)
    dx, dwg, dwu, dwd = ops.gated_mlp_bwd(go, x, None, wg, wu, wd, gk, sg, uk, su, ff.ACTIVATIONS[act], True, True, True)
    g, up = kept64(gk, sg, h), kept64(uk, su, h)
    a, slope, rel = act64(act, g)
    dh, ed = product(go.double(), wd.double().t())
    stored = lambda ref, off: off * (1 + u) + u * ref.abs() + TINY  # noqa: E731
    h64, du, dg = a * up, dh * a, dh * up * slope
    eh = stored(h64, (rel * a.abs() + ACC) * up.abs() + ACC * h64.abs())
    eu = stored(du, ed * a.abs() + dh.abs() * (rel * a.abs() + ACC) + ACC * du.abs())
    slope_off = rel * slope.abs().clamp(min=0.01) + ACC
    eg = stored(dg, (ed * slope.abs() + (ed + dh.abs()) * slope_off) * up.abs() + 2 * ACC * dg.abs())
    close(dwd, *product(h64.t(), go.double(), ea=eh.t()), u, "dw_down")
    close(dwg, *product(x.double().t(), dg, eb=eg), u, "dw_gate")
    close(dwu, *product(x.double().t(), du, eb=eu), u, "dw_up")
    (r1, o1), (r2, o2) = product(dg, wg.double().t(), ea=eg), product(du, wu.double().t(), ea=eu)
    size = dg.abs() @ wg.double().abs().t() + du.abs() @ wu.double().abs().t()
    close(dx, r1 + r2, o1 + o2 + h * ACC * size, u, "dx")


@pytest.mark.parametrize("shape", [(1, 8, 8, 8), (1, 256, 512, 256), (5, 40, 72, 16), (64, 256, 256, 256), (130, 72, 136, 200),
                                   (257, 328, 520, 328), (700, 1000, 264, 1000), (1500, 128, 1408, 136)])
@pytest.mark.parametrize("dtype", list(U))
def test_gated(shape, dtype):
    gated_case(*shape, dtype, "silu", True, 1)
    gated_case(*shape, dtype, "gelu_tanh", False, 2, (True, True, False))
    gated_case(*shape, dtype, "silu", True, 0, (True, False, True))


@pytest.mark.parametrize("shape", [(100, 72, 264, 4096), (300, 72, 520, 4104), (1000, 136, 264, 8192), (300, 136, 4104, 72),
                                   (1001, 264, 4096, 136), (9001, 264, 136, 72)])
@pytest.mark.parametrize("keep", [1, 2])
@pytest.mark.parametrize("dtype", list(U))
def test_gated_long_reductions(shape, keep, dtype):
    """Of the gate's backward, of dx over both projections, and of dw, some in the kernel for few rows, some in shares."""
    gated_case(*shape, dtype, "silu", True, keep)
    gated_case(*shape, dtype, "softplus", False, keep, (False, True, True))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("keep", [1, 2])
@pytest.mark.parametrize("dtype", list(U))
def test_gated_activations(act, keep, dtype):
    gated_case(300, 192, 328, 192, dtype, act, True, keep)


# ------------------------------------------------------------ checkpoints
def checkpoint64(x):
    rows, width = x.shape
    groups = -(-width // 128)
    b = torch.nn.functional.pad(x.double(), (0, groups * 128 - width)).view(rows, groups, 128)
    most = b.abs().amax(-1)
    m, e = torch.frexp(most / 448)
    scale = torch.where(most > 0, torch.ldexp(torch.ones_like(most), torch.where(m > 0.5, e, e - 1)), 0.0).clamp(min=2.0 ** -126)
    y = b / scale[..., None]
    _, e = torch.frexp(y)
    unit = torch.ldexp(torch.ones_like(y), (e - 4).clamp(min=-9))
    return (torch.round(y / unit) * unit).view(rows, -1)[:, :width], scale


@pytest.mark.parametrize("width", [1, 2, 7, 8, 24, 100, 127, 128, 129, 136, 256, 1000, 1999, 4096, 5121])
@pytest.mark.parametrize("dtype", [*U, torch.float32])
def test_checkpoint_to_the_bit(width, dtype):
    """A power of two as the scale: every step but the rounding to 8 bits is exact."""
    for rows in (1, 37):
        x = make(rows, width, dtype=dtype, seed=7) * torch.logspace(-4, 3, rows, device="cuda")[:, None].to(dtype)
        x[0, : width // 2] = 0
        x[rows // 2] = 0
        q, scale = fp8_checkpoint(x)
        want, s = checkpoint64(x)
        assert q.dtype == FP8 and q.shape == x.shape and torch.equal(scale.double(), s) and torch.equal(q.double(), want)
        for t in (*U, torch.float32):
            most = torch.finfo(t).max
            back = fp8_restore(q, scale, t)
            assert torch.equal(back, (want * s.repeat_interleave(128, dim=1)[:, :width]).clamp(-most, most).to(t))


@pytest.mark.parametrize("width", [128, 200, 1999])
def test_checkpoint_borders(width):
    """Largest magnitudes next to 448 times a power of two, the type's largest and smallest values, infinities and NaN."""
    for top in (448.0, 448.0 * (1 + 2.0 ** -23), 448.0 * (1 - 2.0 ** -24), 3.4028234e38, 1e-45, 1.1754944e-38, 2.0 ** -118 * 1.76):
        x = make(3, width, dtype=torch.float32, seed=8, scale=1e-3) * top
        x[:, -1] = torch.tensor([top, -top, top / 2])
        q, scale = fp8_checkpoint(x)
        want, s = checkpoint64(x)
        assert torch.equal(scale.double(), s) and torch.equal(q.double(), want)
        assert torch.isfinite(fp8_restore(q, scale, torch.float32)).all()
    x = make(4, width, dtype=torch.float16, seed=9)
    x[0, 0], x[1, width // 2], x[3, -1] = float("inf"), float("nan"), 65504.0
    back = fp8_restore(*fp8_checkpoint(x), torch.float16)
    groups = torch.arange(width, device="cuda") // 128
    assert torch.isnan(back[0, groups == 0]).all() and torch.isfinite(back[0, groups != 0]).all()
    assert torch.isnan(back[1, groups == width // 2 // 128]).all() and torch.isfinite(back[2:]).all()
    assert back[3, -1] == 65504.0


# ------------------------------------------------------------ autograd
def leaves(*ts):
    return [t.detach().clone().requires_grad_() for t in ts]


@pytest.mark.parametrize("fp8", [False, True])
def test_autograd_is_the_operators(fp8):
    dtype = torch.bfloat16
    x, w, b, r = leaves(make(5, 60, 136, dtype=dtype, seed=1), make(136, 264, dtype=dtype, seed=2, scale=0.1),
                        make(264, dtype=torch.float32, seed=3), make(5, 60, 264, dtype=dtype, seed=4))
    go = make(5, 60, 264, dtype=dtype, seed=5)
    kept = FP8 if fp8 else None
    out = fused_linear(x, w, b, activation="silu", residual=r, activation_dtype=kept)
    got = torch.autograd.grad(out, (x, w, b, r), go)
    with torch.no_grad():
        want, *z = ops.linear(x, w, b, r, 2, 2 if fp8 else 1)
        saved = ops.fp8_checkpoint(x) if fp8 else (x, None)
        grads = ops.linear_bwd(go, *saved, w, *(z if fp8 else (z[0], None)), 2, torch.float32, True, True, True)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(got, [*grads, go]))
    wg, wu, wd = leaves(make(136, 200, dtype=dtype, seed=6, scale=0.1), make(136, 200, dtype=dtype, seed=7, scale=0.1),
                        make(200, 264, dtype=dtype, seed=8, scale=0.1))
    out = fused_gated_mlp(x, wg, wu, wd, residual=r, activation_dtype=kept)
    got = torch.autograd.grad(out, (x, wg, wu, wd, r), go)
    with torch.no_grad():
        want, *k = ops.gated_mlp(x, wg, wu, wd, r, 2, 2 if fp8 else 1)
        k = k if fp8 else (k[0], None, k[1], None)
        grads = ops.gated_mlp_bwd(go, *saved, wg, wu, wd, *k, 2, True, True, True)
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(got, [*grads, go]))


def test_gradients_of_some_inputs():
    """Each gradient by itself is the one that all together give; an unused output's gradient is none."""
    dtype = torch.float16
    base = [make(70, 72, dtype=dtype, seed=1), make(72, 40, dtype=dtype, seed=2, scale=0.1), make(40, dtype=dtype, seed=3),
            make(70, 40, dtype=dtype, seed=4)]
    go = make(70, 40, dtype=dtype, seed=5)
    for act in (None, "silu"):
        x, w, b, r = leaves(*base)
        want = torch.autograd.grad(fused_linear(x, w, b, activation=act, residual=r), (x, w, b, r), go)
        for i in range(4):
            one = [t.detach().requires_grad_(k == i) for k, t in enumerate(base)]
            got, = torch.autograd.grad(fused_linear(*one[:3], activation=act, residual=one[3]), one[i], go)
            assert torch.equal(got, want[i])
    base = [base[0], make(72, 48, dtype=dtype, seed=6, scale=0.1), make(72, 48, dtype=dtype, seed=7, scale=0.1),
            make(48, 40, dtype=dtype, seed=8, scale=0.1), base[3]]
    all_ = leaves(*base)
    want = torch.autograd.grad(fused_gated_mlp(*all_[:4], residual=all_[4]), all_, go)
    for i in range(5):
        one = [t.detach().requires_grad_(k == i) for k, t in enumerate(base)]
        got, = torch.autograd.grad(fused_gated_mlp(*one[:4], residual=one[4]), one[i], go)
        assert torch.equal(got, want[i])


@pytest.mark.parametrize("op", ["linear", "gated"])
def test_gradient_against_differences(op):
    """<grad, d> against central differences of the 64-bit formula along d, step 1e-4 (error 1e-7 or so): the 16-bit
    operands and gradients are off by 2^-11 each, in sums of random signs; 1 % of the norms' product covers them."""
    dtype = torch.float16
    x, ws = make(40, 64, dtype=dtype, seed=1), [make(64, 96, dtype=dtype, seed=2, scale=0.2)]
    if op == "gated":
        ws += [make(64, 96, dtype=dtype, seed=3, scale=0.2), make(96, 64, dtype=dtype, seed=4, scale=0.2)]
        own = lambda x, *w: fused_gated_mlp(x, *w, activation="gelu_tanh")  # noqa: E731
        ref = lambda x, g, u, d: (act64("gelu_tanh", x @ g)[0] * (x @ u)) @ d  # noqa: E731
    else:
        own = lambda x, w: fused_linear(x, w, activation="softplus")  # noqa: E731
        ref = lambda x, w: act64("softplus", x @ w)[0]  # noqa: E731
    args = leaves(x, *ws)
    out = own(*args)
    go = make(*out.shape, dtype=dtype, seed=5)
    for k, (leaf, grad) in enumerate(zip(args, torch.autograd.grad(out, args, go))):
        d = make(*leaf.shape, dtype=torch.float64, seed=10 + k)
        wide = [t.detach().double() for t in args]
        ends = []
        for sign in (1, -1):
            moved = list(wide)
            moved[k] = moved[k] + sign * 1e-4 * d
            ends.append((ref(*moved) * go.double()).sum())
        slope = ((ends[0] - ends[1]) / 2e-4).item()
        assert abs((grad.double() * d).sum().item() - slope) <= 0.01 * (grad.double().norm() * d.norm()).item()
