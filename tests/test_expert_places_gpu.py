"""Plans that no sort gave: places outside the rows, and more rows kept than there
are.  Nothing is read or written there, and the other slots are as always."""
import pytest
import torch

from mlp_megakernel_b200 import ExpertPlan, expert_combine, expert_dispatch

pytestmark = pytest.mark.gpu


def randn(*shape, dtype, seed):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("top", [1, 2, 3, 8])
@pytest.mark.parametrize("width", [24, 33, 258, 2048, 5000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("kept", [-5, 0, 40, 2 ** 31 - 1])
def test_places_outside_the_rows(top, width, dtype, kept):
    tokens = 50
    slots = tokens * top
    g = torch.Generator(device="cuda").manual_seed(top)
    row_of = torch.randperm(slots, device="cuda", generator=g).int()
    bad = torch.rand(slots, device="cuda", generator=g) < 0.3
    row_of[bad] = torch.tensor([-1, -2 ** 31, slots, slots + 1, 2 ** 31 - 1], device="cuda", dtype=torch.int64)[
        torch.arange(int(bad.sum()), device="cuda") % 5].int()
    row_of, bad = row_of.view(tokens, top), bad.view(tokens, top)
    plan = ExpertPlan(row_of, torch.tensor([0, kept], device="cuda", dtype=torch.int32))
    on = ~bad & (row_of < min(max(kept, 0), slots))
    at = torch.where(bad, 0, row_of).long()
    x, y = randn(tokens, width, dtype=dtype, seed=1).requires_grad_(), randn(slots, width, dtype=dtype, seed=2).requires_grad_()
    w = torch.rand(tokens, top, device="cuda", requires_grad=True)
    xs = expert_dispatch(x, plan)
    assert torch.equal(xs[at[on]], x[:, None].expand(-1, top, -1)[on])
    assert not xs[at[~bad & ~on]].any()
    out = expert_combine(y, w, plan)
    terms = torch.where(on[:, :, None], w[:, :, None].double() * y[at].double(), 0.0)
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    room = u * terms.sum(1).abs() + (top + 1) * 2.0 ** -24 * terms.abs().sum(1) + 2.0 ** -25
    assert ((out.double() - terms.sum(1)).abs() <= room).all()
    gout, gxs = randn(tokens, width, dtype=dtype, seed=3), randn(slots, width, dtype=dtype, seed=4)
    dx, dy, dw = torch.autograd.grad((xs, out), (x, y, w), (gxs, gout))
    terms = torch.where(on[:, :, None], gxs[at].double(), 0.0)
    room = u * terms.sum(1).abs() + (top + 1) * 2.0 ** -24 * terms.abs().sum(1) + 2.0 ** -25
    assert ((dx.double() - terms.sum(1)).abs() <= room).all()
    want = w.detach()[:, :, None].double() * gout.double()[:, None]
    assert ((dy[at[on]].double() - want[on]).abs() <= (u + 2.0 ** -24) * want[on].abs() + 2.0 ** -25).all()
    assert not dy[at[~bad & ~on]].any()
    terms = y[at].double() * gout.double()[:, None]
    room = (min(width, 1024) + 13) * 2.0 ** -24 * terms.abs().sum(2) + 2.0 ** -25
    assert ((dw.double() - terms.sum(2)).abs()[on] <= room[on]).all() and not dw[~on].any()
