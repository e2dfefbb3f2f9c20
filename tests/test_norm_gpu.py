"""RMS norm with the residual's addition, its 8-bit output and its gradients
against the formulas in 64 bits.

Tolerances.  u is the unit roundoff of the output's type (2^-11 fp16, 2^-8
bf16, 2^-24 fp32) and w = 2^-24 that of the arithmetic.  The sum of squares has
positive terms, added in runs of at most 64 and trees: a relative error of at
most 100 w, half of that in its root; the products add 4 w.  So
|y - ref| <= (u + 60 w) |ref| + 2^-25 (half of fp16's smallest step).
"""
import math

import pytest
import torch

from mlp_megakernel_b200 import FusedRMSNorm, fused_rms_norm, fused_rms_norm_fp8

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
W = 2.0 ** -24
EPS = 1e-6
WIDTHS = [1, 2, 7, 8, 24, 33, 64, 127, 128, 129, 256, 257, 520, 1000, 1023, 1024, 1032, 2050, 4096, 5120, 8193, 16384,
          32767, 32768]


def make(rows, width, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(rows, width, device="cuda", generator=g)).to(dtype)


def reference(x, w, r, eps=EPS):
    h = x.double() if r is None else x.double() + r.double()
    s = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h, s, h * s if w is None else h * s * w.double()


def close(got, ref, rel, absolute=2.0 ** -25):
    off = (got.double() - ref).abs() - (rel * ref.abs() + absolute)
    assert off.max().item() <= 0 if off.numel() else True, f"off by {off.max().item()} more than allowed"


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", list(U))
def test_forward(width, dtype):
    for rows, residual, weight in ((1, True, dtype), (5, False, None), (67, True, torch.float32)):
        x, r = make(rows, width, dtype, 1), make(rows, width, dtype, 2, 3.0) if residual else None
        w = None if weight is None else (1 + 0.1 * make(1, width, torch.float32, 3)[0]).to(weight)
        got = fused_rms_norm(x, w, residual=r, eps=EPS)
        y, h = got if residual else (got, None)
        ref_h, _, ref = reference(x, w, r)
        close(y, ref, U[dtype] + 60 * W)
        if residual:
            assert torch.equal(h, ref_h.to(torch.float32).to(dtype))  # two values of the type: one rounding to fp32


@pytest.mark.parametrize("width", [1, 8, 33, 127, 128, 129, 256, 300, 1000, 1032, 2050, 5120, 8193, 16384, 32767])
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("dtype", list(U))
def test_fp8(width, group, dtype):
    """scale as max|y| / 448 (as exact as y); q within half a step of e4m3 of
    y / scale: 2^-4 of the value, or 2^-10 below the smallest normal number."""
    for rows, residual in ((1, True), (37, False)):
        x, r = make(rows, width, dtype, 4), make(rows, width, dtype, 5) if residual else None
        x[0, : width // 2] = 0
        w = (1 + 0.1 * make(1, width, torch.float32, 6)[0]).to(dtype)
        with torch.no_grad():
            q, scale, *h = fused_rms_norm_fp8(x, w, residual=r, eps=EPS, group=group)
        _, _, ref = reference(x, w, r)
        g = group or width
        groups = -(-width // g)
        assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and scale.shape == (rows, groups)
        padded = torch.nn.functional.pad(ref, (0, groups * g - width)).view(rows, groups, g)
        close(scale, padded.abs().amax(-1) / 448, 64 * W, 0.0)
        each = scale.double().repeat_interleave(g, dim=1)[:, :width]
        off = (q.double() * each - ref).abs() - (ref.abs() * (2.0 ** -4 + 64 * W) + each * 2.0 ** -10)
        assert off.max().item() <= 0
        if residual:
            assert torch.equal(h[0], (x.double() + r.double()).to(torch.float32).to(dtype))
        else:
            assert not h


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", list(U))
def test_backward(width, dtype):
    """dx = s (gw - n c) + gh, |error| <= u |dx| + w (110 s (|gw| + |n| mean|gw n|) + |gh|)
    (100 w in s and in c's sum, a few products), dw_j = sum_rows g n with
    |error| <= u |dw| + (rows + 110) w sum|g n|."""
    for rows, residual in ((1, False), (3, True), (300, True)):
        if rows == 300 and width > 9000:
            rows = 40
        x = make(rows, width, dtype, 1).requires_grad_()
        r = make(rows, width, dtype, 2).requires_grad_() if residual else None
        w = (1 + 0.1 * make(1, width, torch.float32, 3)[0]).to(dtype).requires_grad_()
        gy, gh = make(rows, width, dtype, 7), make(rows, width, dtype, 8) if residual else None
        if residual:
            y, h = fused_rms_norm(x, w, residual=r, eps=EPS)
            dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (gy, gh))
            assert torch.equal(dx, dr)
        else:
            dx, dw = torch.autograd.grad(fused_rms_norm(x, w, eps=EPS), (x, w), gy)
        h, s, _ = reference(x.detach(), None, None if r is None else r.detach())
        n, gw = h * s, gy.double() * w.detach().double()
        ref = s * (gw - n * (gw * n).mean(-1, keepdim=True))
        room = 110 * W * s * (gw.abs() + n.abs() * (gw * n).abs().mean(-1, keepdim=True))
        if residual:
            ref, room = ref + gh.double(), room + W * gh.double().abs()
        assert ((dx.double() - ref).abs() - U[dtype] * ref.abs() - room - 2.0 ** -25).max().item() <= 0
        gn = gy.double() * n
        room = (rows + 110) * W * gn.abs().sum(0)
        assert ((dw.double() - gn.sum(0)).abs() - U[dtype] * gn.sum(0).abs() - room - 2.0 ** -25).max().item() <= 0


@pytest.mark.parametrize("rows,width", [(3, 5), (11, 128), (4, 1032)])
def test_gradient_against_differences(rows, width):
    """The derivative along a direction d of the 64-bit forward, by central
    differences with a step of 1e-5 (an error of 1e-8 or so), against <grad, d>
    in fp32: at most 2e-5 of sum |grad d|, and 1e-6 of it absolutely."""
    x, r, w = make(rows, width, torch.float32, 1), make(rows, width, torch.float32, 2), make(1, width, torch.float32, 3)[0]
    gy, gh = make(rows, width, torch.float32, 4), make(rows, width, torch.float32, 5)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = fused_rms_norm(leaves[0], leaves[2], residual=leaves[1], eps=EPS)
    grads = torch.autograd.grad((y, h), leaves, (gy, gh))
    for k, t in enumerate((x, r, w)):
        d = torch.randn_like(t, dtype=torch.float64)

        def loss(e):
            a = [v.double() for v in (x, r, w)]
            a[k] = a[k] + e * d
            hh, _, yy = reference(a[0], a[2], a[1])
            return (yy * gy.double()).sum() + (hh * gh.double()).sum()

        slope = ((loss(1e-5) - loss(-1e-5)) / 2e-5).item()
        along = grads[k].double() * d
        assert abs(along.sum().item() - slope) <= 2e-5 * along.abs().sum().item() + 1e-6


def test_unused_outputs_and_frozen_inputs():
    x, r, w = make(9, 96, torch.float32, 1).requires_grad_(), make(9, 96, torch.float32, 2), torch.ones(96, device="cuda")
    y, h = fused_rms_norm(x, w, residual=r)
    dx, = torch.autograd.grad(h.sum(), x, retain_graph=True)
    assert torch.equal(dx, torch.ones_like(x))
    dx, = torch.autograd.grad((y * h.detach()).sum(), x)
    both, = torch.autograd.grad(sum((t * g).sum() for t, g in zip(fused_rms_norm(x, w, residual=r),
                                                                 (h.detach(), torch.zeros_like(h)))), x)
    assert torch.equal(dx, both)
    wl = w.clone().requires_grad_()
    dw, = torch.autograd.grad(fused_rms_norm(x.detach(), wl).sum(), wl)
    n = reference(x.detach(), None, None)[2]
    assert (dw.double() - n.sum(0)).abs().max().item() <= 120 * W * n.abs().sum(0).max().item()


def test_many_rows_and_repeatable():
    """More rows than one wave of blocks; the gradients are the same bits twice."""
    x = make(70001, 40, torch.float16, 1).requires_grad_()
    w = torch.ones(40, device="cuda", dtype=torch.float16, requires_grad=True)
    g = make(70001, 40, torch.float16, 2, 0.01)
    first = torch.autograd.grad(fused_rms_norm(x, w), (x, w), g)
    again = torch.autograd.grad(fused_rms_norm(x, w), (x, w), g)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    gn = g.double() * reference(x.detach(), None, None)[2]
    room = U[torch.float16] * gn.sum(0).abs() + 1000 * W * gn.abs().sum(0)
    assert ((first[1].double() - gn.sum(0)).abs() - room).max().item() <= 0


@pytest.mark.parametrize("rows,width,dtype", [(1, 1999, torch.float16), (7, 2049, torch.bfloat16), (296, 517, torch.float32),
                                              (592, 2049, torch.bfloat16), (1776, 300, torch.float16),
                                              (148, 8190, torch.float16)])
def test_last_rows_of_ragged_widths(rows, width, dtype):
    """Rows whose next one would begin at the tensor's end: what lies behind the
    tensor (NaN here) is neither read nor used, and nothing is written there."""
    def edged(seed):
        big = torch.full((rows * width + 4096,), math.nan, device="cuda", dtype=dtype)
        big[:rows * width] = make(1, rows * width, dtype, seed)[0]
        return big, big[:rows * width].view(rows, width)

    (_, x), (_, r), (_, gy), (_, gh) = (edged(k) for k in range(4))
    w = torch.ones(width, device="cuda", dtype=dtype, requires_grad=True)
    xl, rl = x.detach().requires_grad_(), r.detach().requires_grad_()
    y, h = fused_rms_norm(xl, w, residual=rl, eps=EPS)
    ref_h, s, ref = reference(x, None, r)
    close(y, ref, U[dtype] + 60 * W)
    dx, dw = torch.autograd.grad((y, h), (xl, w), (gy, gh))
    n, g = ref_h * s, gy.double()
    want = s * (g - n * (g * n).mean(-1, keepdim=True))
    room = 110 * W * s * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) + W * gh.double().abs()
    want = want + gh.double()
    assert ((dx.double() - want).abs() - U[dtype] * want.abs() - room - 2.0 ** -25).max().item() <= 0
    gn = g * n
    assert ((dw.double() - gn.sum(0)).abs() - U[dtype] * gn.sum(0).abs() - (rows + 110) * W * gn.abs().sum(0)
            - 2.0 ** -25).max().item() <= 0
    with torch.no_grad():
        q, scale = fused_rms_norm_fp8(x, group=128)
    assert q.float().isfinite().all() and scale.isfinite().all()


def test_rows_without_values():
    for shape in ((0, 64), (3, 0, 128), (0, 7)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w = torch.ones(shape[-1], device="cuda", requires_grad=True)
        y = fused_rms_norm(x, w)
        assert y.shape == shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == shape and torch.equal(dw, torch.zeros_like(w))
        with torch.no_grad():
            q, scale = fused_rms_norm_fp8(x, w, group=128)
        assert q.shape == shape and scale.shape == (*shape[:-1], -(-shape[-1] // 128))


@pytest.mark.parametrize("width", [33, 128, 4096])
def test_zero_and_non_finite_rows(width):
    x = make(6, width, torch.float32, 1)
    x[0] = 0
    x[1, 3] = math.inf
    x[2, 5] = math.nan
    x[3] = 0
    x[3, 1] = 1e-30
    x[4] *= 1e-25  # the 8-bit scale itself is tiny, and eps keeps the row so
    y = fused_rms_norm(x, eps=EPS)
    ref = reference(x, None, None)[2].float()
    assert torch.equal(y[0], torch.zeros_like(y[0]))
    assert torch.equal(y[1].isnan(), ref[1].isnan()) and y[1].nan_to_num().abs().max().item() == 0
    assert y[2].isnan().all()
    close(y[3:], ref[3:].double(), U[torch.float32] + 60 * W, 1e-45)
    for group in (0, 128):
        q, scale = fused_rms_norm_fp8(x, eps=EPS, group=group)
        q, scale = q.float(), scale.repeat_interleave(group or width, dim=1)[:, :width]
        back = q * scale
        assert torch.equal(back[0], torch.zeros_like(back[0])) and scale[0].max().item() == 0
        assert torch.equal(q[1].isnan(), ref[1].isnan()) and back[1][: 4].isnan().all()
        assert back[2].isnan().all()
        assert not back[3:].isnan().any()
        assert ((back[4:] - ref[4:]).abs() <= ref[4:].abs() * (2.0 ** -4 + 64 * W) + scale[4:] * 2.0 ** -10).all()
    tiny = torch.full((2, width), 1e-38, device="cuda")  # max / 448 below the smallest normal number
    q, scale = fused_rms_norm_fp8(tiny, eps=1.0)
    assert not q.float().any() and not scale.any()


@pytest.mark.parametrize("width", [64, 100, 1000])
def test_strides_views_and_streams(width):
    """Inputs that are slices, transposed, off 16-byte boundaries, of more
    dimensions, and used on another stream than the default one."""
    big = make(50, 2 * width + 3, torch.float16, 1)
    x, r = big[:, 3:3 + width], make(width, 50, torch.float16, 2).t()
    w = make(1, width + 1, torch.float16, 3)[0, 1:]
    want = fused_rms_norm(x.contiguous(), w.clone(), residual=r.contiguous())
    for a, b in zip(fused_rms_norm(x, w, residual=r), want):
        assert torch.equal(a, b)
    shaped = fused_rms_norm(x.reshape(5, 10, width), w, residual=r.reshape(5, 10, width))
    assert all(torch.equal(a.view(50, width), b) for a, b in zip(shaped, want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = x.contiguous() * 2
        got = fused_rms_norm(late, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, fused_rms_norm(x.contiguous() * 2, w))


def test_rows_past_32_bits():
    """Elements beyond 2^31 of one tensor: the last rows are right."""
    rows, width = 33000, 65536 // 2
    if torch.cuda.get_device_properties(0).total_memory < 20 << 30:
        pytest.skip("needs 5 GB")
    rows = 2 ** 31 // width + 3000
    x = torch.zeros(rows, width, device="cuda", dtype=torch.float16)
    x[-3:] = make(3, width, torch.float16, 1)
    y = fused_rms_norm(x)
    close(y[-3:], reference(x[-3:], None, None)[2], U[torch.float16] + 60 * W)
    assert not y[-3000:-3].any()


def test_module_and_graph():
    m = FusedRMSNorm(96).cuda()
    x, r = make(10, 96, torch.float32, 1), make(10, 96, torch.float32, 2)
    y, h = m(x, r)
    assert torch.equal(h, x + r) and y.requires_grad
    static = torch.zeros_like(x)
    with torch.no_grad():
        m(static, r)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, _ = m(static, r)
        static.copy_(x)
        g.replay()
    assert torch.equal(out, y)


def test_compiled():
    m = FusedRMSNorm(64).cuda()
    x, r = make(20, 64, torch.float16, 1), make(20, 64, torch.float16, 2)

    def f(a, b):
        y, h = m(a, b)
        return y * 2, h

    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    want, got = f(a, r), torch.compile(f, fullgraph=True)(b, r)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    assert torch.equal(torch.autograd.grad(want[0].sum(), a)[0], torch.autograd.grad(got[0].sum(), b)[0])
