"""Rows that a block comes to after its first: the ring of copies, the halves of
the row sums and the group maxima come round several times, with values that are
other ones in every row.  Formulas and tolerances are those of test_norm_gpu.py
(the row count enters dw's)."""
import pytest
import torch

from mlp_megakernel_b200 import FusedRMSNorm, fused_rms_norm, fused_rms_norm_fp8

from .test_norm_gpu import EPS, U, W, close, make, reference

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
# At least 7 rows for each block (or row group of a block) that 148 SMs can hold
# by their threads alone: two more than the ring has.
CASES = [
    (8300, 4096, BF16), (16600, 1024, F32), (4200, 16384, BF16), (2100, 16384, F32),  # every thread all its vectors
    (133000, 128, F16), (66400, 800, F16), (22000, 1032, F16), (66400, 264, F32),     # some have fewer
    (266000, 33, BF16), (24900, 517, F32), (16600, 1999, F16), (16600, 2049, BF16), (7300, 8191, F16),  # ragged
]


def rows_of(rows, width, dtype, seed):
    """Normal values, each row of another size."""
    t = make(rows, width, F32, seed)
    t *= 0.25 + make(rows, 1, F32, seed + 1000).abs()
    return t.to(dtype)


@pytest.mark.parametrize("rows,width,dtype", CASES)
@pytest.mark.parametrize("residual", [False, True])
def test_forward(rows, width, dtype, residual):
    x, r = rows_of(rows, width, dtype, 1), rows_of(rows, width, dtype, 2) if residual else None
    w = (1 + 0.1 * make(1, width, F32, 3)[0]).to(dtype)
    got = fused_rms_norm(x, w, residual=r, eps=EPS)
    y, h = got if residual else (got, None)
    for a in range(0, rows, 20000):  # the reference in parts
        part = slice(a, a + 20000)
        ref_h, _, ref = reference(x[part], w, r[part] if residual else None)
        close(y[part], ref, U[dtype] + 60 * W)
        if residual:
            assert torch.equal(h[part], ref_h.float().to(dtype))


@pytest.mark.parametrize("rows,width,dtype", CASES)
@pytest.mark.parametrize("group", [0, 128])
def test_fp8(rows, width, dtype, group):
    x, r = rows_of(rows, width, dtype, 4), rows_of(rows, width, dtype, 5)
    w = (1 + 0.1 * make(1, width, F32, 6)[0]).to(dtype)
    g = group or width
    groups = -(-width // g)
    for residual in (r, None):
        q, scale, *h = fused_rms_norm_fp8(x, w, residual=residual, eps=EPS, group=group)
        for a in range(0, rows, 20000):
            part = slice(a, a + 20000)
            ref_h, _, ref = reference(x[part], w, None if residual is None else residual[part])
            n = len(ref)
            padded = torch.nn.functional.pad(ref, (0, groups * g - width)).view(n, groups, g)
            close(scale[part], padded.abs().amax(-1) / 448, 64 * W, 0.0)
            each = scale[part].double().repeat_interleave(g, dim=1)[:, :width]
            off = (q[part].double() * each - ref).abs() - (ref.abs() * (2.0 ** -4 + 64 * W) + each * 2.0 ** -10)
            assert off.max().item() <= 0
            if h:
                assert torch.equal(h[0][part], ref_h.float().to(dtype))


def check_backward(x, w, r, gy, gh, dx, dw):
    rows, dtype = len(x), x.dtype
    total = torch.zeros(x.shape[1], device="cuda", dtype=torch.float64)
    spread = torch.zeros_like(total)
    for a in range(0, rows, 20000):
        part = slice(a, a + 20000)
        h, s, _ = reference(x[part], None, None if r is None else r[part])
        g = gy[part].double()
        n, gw = h * s, g if w is None else g * w.double()
        ref = s * (gw - n * (gw * n).mean(-1, keepdim=True))
        room = 110 * W * s * (gw.abs() + n.abs() * (gw * n).abs().mean(-1, keepdim=True))
        if gh is not None:
            ref, room = ref + gh[part].double(), room + W * gh[part].double().abs()
        assert ((dx[part].double() - ref).abs() - U[dtype] * ref.abs() - room - 2.0 ** -25).max().item() <= 0
        total += (g * n).sum(0)
        spread += (g * n).abs().sum(0)
    if dw is not None:
        assert ((dw.double() - total).abs() - U[dw.dtype] * total.abs() - (rows + 110) * W * spread
                - 2.0 ** -25).max().item() <= 0


@pytest.mark.parametrize("rows,width,dtype", CASES)
@pytest.mark.parametrize("residual", [False, True])
def test_backward(rows, width, dtype, residual):
    x = rows_of(rows, width, dtype, 1).requires_grad_()
    r = rows_of(rows, width, dtype, 2).requires_grad_() if residual else None
    # a gradient that is small enough for dw to stay within fp16
    gy, gh = rows_of(rows, width, dtype, 7) * 0.01, rows_of(rows, width, dtype, 8) if residual else None
    w = (1 + 0.1 * make(1, width, F32, 3)[0]).to(dtype).requires_grad_()
    got = fused_rms_norm(x, w, residual=r, eps=EPS)
    if residual:
        dx, dr, dw = torch.autograd.grad(got, (x, r, w), (gy, gh))
        assert torch.equal(dx, dr)
    else:
        dx, dw = torch.autograd.grad(got, (x, w), gy)
    with torch.no_grad():
        check_backward(x, w, r, gy, gh, dx, dw)


@pytest.mark.parametrize("width", [1, 24, 127, 256, 517, 1000, 2050, 4096, 8193, 16384, 32767])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [1, 300])
def test_gradients_of_the_module(rows, width, dtype):
    """16-bit rows with the module's fp32 weight, and with no weight."""
    m = FusedRMSNorm(width, eps=EPS).cuda()
    with torch.no_grad():
        m.weight += 0.1 * make(1, width, F32, 3)[0]
    x, r = make(rows, width, dtype, 1).requires_grad_(), make(rows, width, dtype, 2).requires_grad_()
    gy, gh = make(rows, width, dtype, 7), make(rows, width, dtype, 8)
    dx, dr, dw = torch.autograd.grad(m(x, r), (x, r, m.weight), (gy, gh))
    assert torch.equal(dx, dr) and dw.dtype == F32
    alone, = torch.autograd.grad(fused_rms_norm(x, eps=EPS), x, gy)
    with torch.no_grad():
        check_backward(x, m.weight, r, gy, gh, dx, dw)
        check_backward(x, None, None, gy, None, alone, None)
