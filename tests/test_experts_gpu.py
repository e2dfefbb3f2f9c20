"""Rows sorted by expert and back against index arithmetic and the formulas in
64 bits.

Tolerances.  u is the unit roundoff of the output's type and w = 2^-24 that of
the sums.  combine: K products and sums in fp32: |error| <= u |ref| +
(K + 1) w sum|w y| + 2^-25.  dy: one product, u |ref| + w |ref| + 2^-25.  dw: a
sum over the columns in runs of at most 1024 and trees: u |ref| +
(min(D, 1024) + 12) w sum|g y|.
"""
import numpy as np
import pytest
import torch

from mlp_megakernel_b200 import (ExpertPlan, FusedAdamW, FusedMLPExperts, expert_combine, expert_dispatch, expert_sort)

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
W = 2.0 ** -24


def randn(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def some_ids(tokens, top, experts, seed=0, dtype=torch.int64, drop=0.2):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, experts, (tokens, top))
    skew = rng.random((tokens, top)) < 0.3
    ids[skew] = 0  # one expert that is liked best
    bad = rng.random((tokens, top)) < drop
    ids[bad] = rng.choice([-1, experts, experts + 7, -(2 ** 31)], bad.sum())
    return torch.from_numpy(ids).to("cuda", dtype)


def check_plan(ids, experts, plan):
    flat = ids.cpu().numpy().reshape(-1)
    key = np.where((flat >= 0) & (flat < experts), flat, experts)
    order = np.argsort(key, kind="stable")
    row = np.empty(len(flat), np.int64)
    row[order] = np.arange(len(flat))
    assert np.array_equal(plan.row_of.cpu().numpy().reshape(-1), row)
    first = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=experts + 1))[:experts]])
    assert np.array_equal(plan.offsets.cpu().numpy(), first)
    assert plan.num_experts == experts


@pytest.mark.parametrize("slots", [0, 1, 31, 32, 33, 255, 256, 257, 2049, 5000, 37888, 37889, 300007])
@pytest.mark.parametrize("experts", [1, 2, 8, 37, 255, 256, 257, 1024])
def test_sort(slots, experts):
    for dtype, drop in ((torch.int64, 0.2), (torch.int32, 0.0)):
        ids = some_ids(slots, 1, experts, slots + experts, dtype, drop)
        check_plan(ids, experts, expert_sort(ids, experts))


def test_sort_extremes():
    every = torch.full((4000, 3), 5, device="cuda")
    check_plan(every, 9, expert_sort(every, 9))
    none = torch.full((4000, 3), -1, device="cuda")
    check_plan(none, 9, expert_sort(none, 9))
    wide = torch.tensor([[2 ** 32, 1, -(2 ** 40)]], device="cuda")  # not expert 0 after a cut to 32 bits
    check_plan(wide, 2, expert_sort(wide, 2))
    ids = some_ids(3, 500, 7, 1).t()  # strided
    check_plan(ids, 7, expert_sort(ids, 7))
    check_plan(ids[1:], 7, expert_sort(ids[1:], 7))
    big = some_ids(2_200_000, 2, 300, 3, torch.int32)
    check_plan(big, 300, expert_sort(big, 300))


def gathered(t, plan, kept):
    """t's row of each kept slot, zeros for the others: [tokens, choices, width]."""
    at = plan.row_of.long()
    return torch.where(kept[:, :, None], t[at].double(), 0.0)


CASES = [(1, 1, 1, 1), (1, 2, 4, 8), (5, 3, 4, 7), (64, 2, 8, 128), (33, 8, 16, 100), (100, 1, 3, 257), (7, 6, 64, 1032),
         (513, 2, 5, 24), (40, 4, 16, 4096), (3, 2, 4, 16384), (70, 9, 12, 66), (2000, 2, 1024, 16)]


@pytest.mark.parametrize("tokens,top,experts,width", CASES)
@pytest.mark.parametrize("dtype", list(U))
def test_dispatch_and_combine(tokens, top, experts, width, dtype):
    for drop, w_dtype in ((0.0, torch.float32), (0.3, dtype), (1.0, None)):
        ids = some_ids(tokens, top, experts, 5, drop=drop)
        plan = expert_sort(ids, experts)
        kept = plan.row_of < plan.offsets[-1]
        x, y = randn(tokens, width, dtype=dtype, seed=1), randn(tokens * top, width, dtype=dtype, seed=2)
        y[int(plan.offsets[-1]):] = float("nan")  # what is in a dropped slot's row is not looked at
        w = None if w_dtype is None else torch.softmax(randn(tokens, top, seed=3), 1).to(w_dtype)
        if w is not None:
            w[~kept] = float("nan")
        x.requires_grad_()
        y.requires_grad_()
        if w is not None:
            w.requires_grad_()
        xs, out = expert_dispatch(x, plan), expert_combine(y, w, plan)
        want = torch.zeros_like(xs)
        at = plan.row_of.long()
        want[at[kept]] = x.detach()[:, None, :].expand(-1, top, -1)[kept]
        assert torch.equal(xs, want)
        wk = torch.where(kept, 1.0 if w is None else w.detach().double(), 0.0)
        ys = gathered(y.detach(), plan, kept)
        terms = wk[:, :, None] * ys
        room = (top + 1) * W * terms.abs().sum(1) + 2.0 ** -25
        ref = terms.sum(1)
        assert ((out.double() - ref).abs() - U[dtype] * ref.abs() - room).max().item() <= 0

        gxs, g = randn(tokens * top, width, dtype=dtype, seed=6), randn(tokens, width, dtype=dtype, seed=7)
        gxs[int(plan.offsets[-1]):] = float("nan")
        dx, = torch.autograd.grad(xs, x, gxs)
        terms = gathered(gxs, plan, kept)
        room = (top + 1) * W * terms.abs().sum(1) + 2.0 ** -25
        assert ((dx.double() - terms.sum(1)).abs() - U[dtype] * terms.sum(1).abs() - room).max().item() <= 0
        dy, *dw = torch.autograd.grad(out, [y] if w is None else [y, w], g)
        ref = torch.zeros(tokens * top, width, device="cuda", dtype=torch.float64)
        ref[at.view(-1)] = (wk[:, :, None] * g.double()[:, None, :]).view(-1, width)
        assert ((dy.double() - ref).abs() - (U[dtype] + W) * ref.abs() - 2.0 ** -25).max().item() <= 0
        if w is not None:
            terms = ys * g.double()[:, None, :]
            ref, room = terms.sum(2), (min(width, 1024) + 12) * W * terms.abs().sum(2) + 2.0 ** -25
            assert ((dw[0].double() - ref).abs() - U[w_dtype] * ref.abs() - room).max().item() <= 0
            assert not dw[0][~kept].any()


def test_gradient_against_differences():
    """combine is linear in y and in weights: a whole step along a direction
    gives the derivative up to the rounding, 1e-5 of the sum of the magnitudes."""
    plan = expert_sort(some_ids(50, 3, 6, 1), 6)
    y, w, g = randn(150, 40, seed=1), torch.rand(50, 3, device="cuda"), randn(50, 40, seed=2)
    yl, wl = y.clone().requires_grad_(), w.clone().requires_grad_()
    dy, dw = torch.autograd.grad(expert_combine(yl, wl, plan), (yl, wl), g)
    for leaf, grad, at in ((y, dy, 0), (w, dw, 1)):
        d = torch.randn_like(leaf)

        def loss(e):
            args = [y, w]
            args[at] = leaf + e * d
            return (expert_combine(*args, plan).double() * g.double()).sum().item()

        along = (grad.double() * d.double())
        assert abs((loss(0.5) - loss(-0.5)) - along.sum().item()) <= 1e-5 * (g.abs().sum() * 40).item() ** 0.5 + \
            1e-5 * along.abs().sum().item()
    x = randn(50, 40, seed=3).requires_grad_()
    gxs = randn(150, 40, seed=4)
    dx, = torch.autograd.grad(expert_dispatch(x, plan), x, gxs)
    d = torch.randn_like(x)
    slope = ((expert_dispatch(x.detach() + d, plan).double() - expert_dispatch(x.detach(), plan).double()) * gxs).sum()
    along = dx.double() * d.double()
    assert abs(slope.item() - along.sum().item()) <= 1e-5 * along.abs().sum().item() + 1e-4


def test_no_tokens():
    plan = expert_sort(torch.empty(0, 2, device="cuda", dtype=torch.int64), 4)
    assert plan.offsets.tolist() == [0] * 5
    x, y = torch.empty(0, 16, device="cuda", requires_grad=True), torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.empty(0, 2, device="cuda", requires_grad=True)
    xs, out = expert_dispatch(x, plan), expert_combine(y, w, plan)
    assert xs.shape == (0, 16) and out.shape == (0, 16)
    assert [t.shape[0] for t in torch.autograd.grad((xs.sum(), out.sum()), (x, y, w))] == [0, 0, 0]


@pytest.mark.parametrize("width", [12, 64, 4096])
def test_views_and_streams(width):
    ids = some_ids(60, 2, 5, 2)
    plan = expert_sort(ids, 5)
    big, tall = randn(60, width + 5, dtype=torch.float16, seed=1), randn(width, 120, dtype=torch.float16, seed=2)
    x, y, w = big[:, 3:3 + width], tall.t(), torch.rand(2, 61, device="cuda").t()[1:]
    assert torch.equal(expert_dispatch(x, plan), expert_dispatch(x.contiguous(), plan))
    assert torch.equal(expert_combine(y, w, plan), expert_combine(y.contiguous(), w.contiguous(), plan))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = (ids + 1) % 5
        other = expert_sort(late, 5)
        out = expert_combine(expert_dispatch(x, other), w, other)
    torch.cuda.current_stream().wait_stream(s)
    again = expert_sort((ids + 1) % 5, 5)
    assert torch.equal(out, expert_combine(expert_dispatch(x, again), w, again))


def test_rows_past_32_bits():
    """A sorted buffer of more than 2^31 elements."""
    tokens, top, width = 66_000, 2, 16384
    ids = torch.randint(0, 4, (tokens, top), device="cuda")
    plan = expert_sort(ids, 4)
    x = torch.empty(tokens, width, device="cuda", dtype=torch.float16).normal_()
    with torch.no_grad():
        xs = expert_dispatch(x, plan)
        assert torch.equal(xs[plan.row_of[-50:].long()], x[-50:, None].expand(-1, 2, -1))
        out = expert_combine(xs, None, plan)
    assert torch.equal(out[-50:], (x[-50:].float() * 2).half())
    assert torch.equal(out[:50], (x[:50].float() * 2).half())


def test_compiled_and_graph():
    ids, x, w = some_ids(40, 2, 4, 3), randn(40, 32, dtype=torch.float16, seed=1), torch.rand(40, 2, device="cuda")

    def f(ids, x, w):
        plan = expert_sort(ids, 4)
        return expert_combine(expert_dispatch(x, plan) * 2, w, plan)

    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    wa, wb = w.clone().requires_grad_(), w.clone().requires_grad_()
    want, got = f(ids, a, wa), torch.compile(f, fullgraph=True)(ids, b, wb)
    assert torch.equal(want, got)
    for p, q in zip(torch.autograd.grad(want.sum(), (a, wa)), torch.autograd.grad(got.sum(), (b, wb))):
        assert torch.equal(p, q)
    static = torch.zeros_like(ids)
    with torch.no_grad():
        f(static, x, w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f(static, x, w)
        static.copy_(ids)
        graph.replay()
    assert torch.equal(out, want)


@pytest.mark.parametrize("capacity", [None, 20])
def test_block_of_experts(capacity):
    """The module against its parts, one expert at a time; the experts round
    their operands to fp16, so the same calls give nearly the same values."""
    torch.manual_seed(0)
    block = FusedMLPExperts(D=64, H=64, num_experts=4, top=2, capacity=capacity).cuda()
    x, r = randn(90, 64, seed=1).requires_grad_(), randn(90, 64, seed=2)
    out, h = block(x, r)
    y = block.norm(h)
    scores, ids = (y @ block.router).topk(2, dim=1)
    weights = torch.softmax(scores, 1)
    ref = torch.zeros_like(out)
    for e, expert in enumerate(block.experts):
        slot = (ids == e)
        if capacity is not None:
            slot &= (slot.view(-1).cumsum(0) <= capacity).view(slot.shape)
        ref = ref + (weights * slot).sum(1, keepdim=True) * expert(y).float()
    assert (out - ref).abs().max().item() <= 1e-2 * ref.abs().max().item()
    g = randn(90, 64, seed=3)
    params = [x, block.router, block.norm.weight, *block.experts[0].weights]
    for a, b in zip(torch.autograd.grad(out, params, g, retain_graph=True), torch.autograd.grad(ref, params, g)):
        assert (a.double() - b.double()).norm().item() <= 1e-2 * b.double().norm().item()


def test_block_trains_with_the_optimizer():
    """Norm, experts and the 8-bit step together: the loss of a fixed batch falls
    to less than half in 40 steps, and its first steps are the same twice."""
    def run(steps):
        torch.manual_seed(1)
        block = FusedMLPExperts(D=32, H=64, num_experts=4, top=2).cuda()
        opt = FusedAdamW(block.parameters(), lr=3e-3, state_bits=8)
        x = randn(512, 32, seed=1)
        target = torch.sin(2 * x) + x.roll(1, 1)
        losses = []
        for _ in range(steps):
            opt.zero_grad()
            out, h = block(x)
            loss = (out + h - target).square().mean()
            loss.backward()
            opt.step()
            losses.append(loss.item())
        return losses

    losses = run(40)
    assert losses[-1] < 0.5 * losses[0]
    assert run(3) == losses[:3]


def test_plan_is_a_tuple():
    plan = expert_sort(some_ids(10, 2, 3, 1, drop=0.0), 3)
    assert isinstance(plan, ExpertPlan) and plan.counts.sum().item() == 20
