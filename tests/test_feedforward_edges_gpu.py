"""The feed-forward operators at the edges of what their documentation allows:
empty and single rows, layouts, values that are not finite, far offsets, streams,
threads, captured graphs, repeated runs; and a block of them trained together."""
import threading

import pytest
import torch
import torch.nn as nn

from mlp_megakernel_b200 import (FusedAdamW, FusedGatedMLP, FusedLinear, FusedRMSNorm, _lib, fp8_checkpoint, fp8_restore,
                                 fused_gated_mlp, fused_linear)

pytestmark = pytest.mark.gpu
BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def status():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def randn(*shape, seed, dtype=BF16, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


def weights(k=72, h=136, n=40, dtype=BF16):
    return randn(k, h, seed=2, dtype=dtype, scale=0.1), randn(k, h, seed=3, dtype=dtype, scale=0.1), randn(h, n, seed=4, dtype=dtype, scale=0.1)


def grads(out, leaves, go):
    return torch.autograd.grad(out, leaves, go)


@pytest.mark.parametrize("kept", [None, FP8])
def test_no_rows(kept):
    """No output rows; the weights' gradients are zeros."""
    wg, wu, wd = (w.requires_grad_() for w in weights())
    b = torch.zeros(136, device="cuda", requires_grad=True)
    for shape in ((0, 72), (3, 0, 72)):
        x = torch.empty(*shape, device="cuda", dtype=BF16, requires_grad=True)
        out = fused_linear(x, wg, b, activation="silu", activation_dtype=kept)
        assert out.shape == (*shape[:-1], 136)
        got = grads(out, (x, wg, b), torch.empty_like(out))
        assert got[0].shape == x.shape and not got[1].any() and not got[2].any()
        out = fused_gated_mlp(x, wg, wu, wd, activation_dtype=kept)
        got = grads(out, (x, wg, wu, wd), torch.empty_like(out))
        assert out.shape == (*shape[:-1], 40) and all(not g.any() for g in got)
    q, scale = fp8_checkpoint(torch.empty(0, 130, device="cuda"))
    assert q.shape == (0, 130) and scale.shape == (0, 2) and fp8_restore(q, scale).shape == (0, 130)


def test_a_row_without_leading_dimensions():
    x, (wg, wu, wd) = randn(72, seed=1), weights()
    assert torch.equal(fused_linear(x, wg), fused_linear(x[None], wg)[0])
    assert torch.equal(fused_gated_mlp(x, wg, wu, wd), fused_gated_mlp(x[None], wg, wu, wd)[0])
    q, s = fp8_checkpoint(x)
    assert s.shape == (1,) and torch.equal(fp8_restore(q, s), fp8_restore(*fp8_checkpoint(x[None]))[0])


@pytest.mark.parametrize("rows", [3, 200, 700])
def test_layouts(rows):
    """Strided rows, weights as transposes and as slices, pointers off the 16-byte grid: the values of the plain layout."""
    x, r, go = randn(rows, 72, seed=1), randn(rows, 136, seed=5), randn(rows, 136, seed=6)
    w, wu, wd = weights()

    def off(t):  # the same values two bytes off
        buf = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)

    def spread(t):
        wide = torch.zeros(t.shape[0], 2 * t.shape[1], device="cuda", dtype=t.dtype)
        wide[:, : t.shape[1]] = t
        return wide[:, : t.shape[1]]

    def transposed(t):
        return t.t().contiguous().t()

    want = fused_linear(x, w, activation="silu", residual=r)
    for f in (off, spread, transposed):
        assert torch.equal(fused_linear(f(x), f(w), activation="silu", residual=f(r)), want)
    wanted = None
    for f in (lambda t: t, off, spread, transposed):
        a, b = f(x).detach().requires_grad_(), f(w).detach().requires_grad_()
        out = fused_linear(a, b, activation="silu", residual=r)
        got = grads(out, (a, b), f(go))
        wanted = wanted or got
        # x^T dz as (dz^T x)^T is another tiling of the same sums
        close = got[1].float() - wanted[1].float()
        assert torch.equal(got[0], wanted[0]) and close.abs().max() <= 2 ** -7 * wanted[1].float().abs().max()
    base = fused_gated_mlp(x, w, wu, wd)
    assert torch.equal(fused_gated_mlp(x, transposed(w), transposed(wu), wd), base)
    assert torch.equal(fused_gated_mlp(x, transposed(w), wu, transposed(wd)), base)


@pytest.mark.parametrize("rows", [5, 150, 600])
@pytest.mark.parametrize("kept", [None, FP8])
def test_a_row_that_is_not_finite_stays_by_itself(rows, kept):
    x, (wg, wu, wd), go = randn(rows, 72, seed=1), weights(), randn(rows, 40, seed=7)
    bad = x.clone()
    bad[2] = float("nan")
    bad[3, 5] = float("inf")
    rest = [i for i in range(rows) if i not in (2, 3)]
    for f in (lambda t: fused_linear(t, wg, activation="gelu_tanh", activation_dtype=kept),
              lambda t: fused_gated_mlp(t, wg, wu, wd, activation_dtype=kept)):
        a, b = x.clone().requires_grad_(), bad.clone().requires_grad_()
        ya, yb = f(a), f(b)
        assert torch.equal(ya[rest], yb[rest]) and torch.isnan(yb[2]).all() and not torch.isfinite(yb[3]).all()
        g = go if ya.shape[1] == 40 else randn(rows, 136, seed=8)
        (da,), (db,) = grads(ya, (a,), g), grads(yb, (b,), g)
        assert torch.equal(da[rest], db[rest]) and torch.isnan(db[2]).all()


@pytest.mark.parametrize("rows", [5, 150, 600])
def test_a_column_that_is_not_finite_stays_by_itself(rows):
    x, (wg, wu, _) = randn(rows, 72, seed=1), weights()
    bad = wg.clone()
    bad[3, 11] = float("nan")
    keep = [c for c in range(136) if c != 11]
    for act in (None, "relu", "silu", "gelu_tanh", "softplus", "sigmoid"):
        a, b = fused_linear(x, wg, activation=act), fused_linear(x, bad, activation=act)
        assert torch.equal(a[:, keep], b[:, keep]) and torch.isnan(b[:, 11]).all()


def test_far_offsets():
    """Outputs, kept values and checkpoints past 2^31 elements: the last rows are what they are alone."""
    rows, n = 66001, 32768
    x, w, b = randn(rows, 8, seed=1), randn(8, n, seed=2), randn(n, seed=3)
    last = x[-300:].clone()
    with torch.no_grad():
        out = fused_linear(x, w, b, activation="relu")
        assert torch.equal(out[-300:], fused_linear(last, w, b, activation="relu"))
        q, scale = fp8_checkpoint(out)
        want = fp8_checkpoint(out[-300:].contiguous())
        assert torch.equal(q[-300:].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scale[-300:], want[1])
        del out
        back = fp8_restore(q, scale, BF16)
        assert torch.equal(back[-300:], fp8_restore(*want, BF16))
        del back, q
        for keep in (1, 2):
            out, *kept = torch.ops.mlpk.linear(x, w, b, None, 2, keep)
            _, *wanted = torch.ops.mlpk.linear(last, w, b, None, 2, keep)
            for a, c in zip(kept, wanted):
                a, c = a[-300:], c
                assert torch.equal(a.view(torch.uint8) if a.dtype == FP8 else a, c.view(torch.uint8) if c.dtype == FP8 else c)
            del out, kept


def step(x, ws, go, kept=None):
    leaves = [t.detach().requires_grad_() for t in (x, *ws)]
    out = fused_gated_mlp(*leaves, residual=None, activation_dtype=kept)
    return [out.detach(), *grads(out, leaves, go)]


@pytest.mark.parametrize("rows,k,h", [(7, 72, 136), (300, 264, 520), (3000, 256, 1032)])
@pytest.mark.parametrize("kept", [None, FP8])
def test_the_same_bits_every_time_and_from_graphs(rows, k, h, kept):
    """Repeated runs, a captured and replayed step (new inputs in the same buffers), two graphs of one step."""
    x, go, ws = randn(rows, k, seed=1), randn(rows, 40, seed=5), weights(k, h)
    first = step(x, ws, go, kept)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(step(x, ws, go, kept), first))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x, ws, go, kept))
        graphs.append(g)
    x2 = randn(rows, k, seed=11)
    want = step(x2, ws, go, kept)
    x.copy_(x2)
    for _ in range(2):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_other_streams_and_threads():
    """Calls on several streams and host threads at once, each with its own inputs."""
    cases = [(randn(rows, 264, seed=rows), randn(rows, 40, seed=rows + 1)) for rows in (3, 150, 700, 2500)]
    ws = weights(264, 520)
    want = [step(x, ws, go) for x, go in cases]
    torch.cuda.synchronize()
    got, errors = [None] * len(cases), []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got[i] = step(cases[i][0], ws, cases[i][1])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_the_same_tensor_in_several_places():
    """x as its own residual, one weight for gate and partner: gradients are the sums of both places'."""
    x, (wg, _, _), go = randn(90, 72, seed=1, dtype=F16), weights(dtype=F16), randn(90, 72, seed=2, dtype=F16)
    wd = randn(136, 72, seed=9, dtype=F16, scale=0.1)
    a, w = x.clone().requires_grad_(), wg.clone().requires_grad_()
    dx, dw = grads(fused_gated_mlp(a, w, w, wd, residual=a), (a, w), go)
    p = [t.clone().requires_grad_() for t in (x, wg, wg, x)]
    each = grads(fused_gated_mlp(p[0], p[1], p[2], wd, residual=p[3]), p, go)
    assert torch.equal(dx, each[0] + each[3]) and torch.equal(dw, each[1] + each[2])


def test_a_saved_input_changed_in_place_is_noticed():
    x, (wg, _, _) = randn(20, 72, seed=1), weights()
    w = wg.requires_grad_()
    out = fused_linear(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


class Block(nn.Module):
    """Norm, gated block with the residual, norm, linear layer with the residual."""

    def __init__(self, width, hidden, kept):
        super().__init__()
        self.n1, self.n2 = FusedRMSNorm(width), FusedRMSNorm(width)
        self.mlp = FusedGatedMLP(width, hidden, activation_dtype=kept)
        self.out = FusedLinear(width, width, activation="gelu_tanh", activation_dtype=kept)

    def forward(self, h):
        h = self.mlp(self.n1(h), residual=h)
        return self.out(self.n2(h), residual=h)


def plain(block, h):
    def norm(m, t):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + m.eps) * m.weight.double()

    y = norm(block.n1, h)
    g, u = y @ block.mlp.w_gate.double(), y @ block.mlp.w_up.double()
    h = h + (torch.nn.functional.silu(g) * u) @ block.mlp.w_down.double()
    z = norm(block.n2, h) @ block.out.weight.double() + block.out.bias.double()
    return h + torch.nn.functional.gelu(z, approximate="tanh")


@pytest.mark.parametrize("kept", [None, FP8])
@pytest.mark.parametrize("autocast", [False, True])
def test_a_block_trains(kept, autocast):
    """Gradients of a block against those of the formula in 64 bits, by their direction: 8 roundings to bf16 (2^-8 of a
    value at most each) on the way leave 3 % of the norm, kept values in 8 bits (2^-4 each, three of them) 15 %.  Then
    steps of the optimizer run."""
    torch.manual_seed(0)
    block = Block(264, 520, kept).cuda()
    opt = FusedAdamW(block.parameters(), lr=1e-3)
    x = randn(400, 264, seed=1, dtype=F32 if autocast else BF16)
    go = randn(400, 264, seed=2, dtype=F32)
    for turn in range(3):
        opt.zero_grad()
        with torch.autocast("cuda", dtype=BF16, enabled=autocast):
            out = block(x)
        out.float().backward(go)
        if turn == 0:
            got = [p.grad.double().clone() for p in block.parameters()]
            wanted = torch.autograd.grad(plain(block, x.double()), list(block.parameters()), go.double())
            for a, b in zip(got, wanted):
                assert (a - b).norm() <= (0.15 if kept else 0.03) * b.norm()
        opt.step()
    assert all(torch.isfinite(p).all() for p in block.parameters())
