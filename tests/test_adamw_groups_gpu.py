"""Parameter groups of FusedAdamW with options of their own, and changed between
steps as torch's optimizers allow it: what is stepped is what the groups hold, and
a parameter keeps its state."""
import pytest
import torch

from mlp_megakernel_b200 import FusedAdamW

pytestmark = pytest.mark.gpu

HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def randn(n, seed):
    return torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def make(sizes, seed=0, dtype=torch.float32):
    params = []
    for k, n in enumerate(sizes):
        p = torch.nn.Parameter(randn(n, seed + k).to(dtype))
        p.grad = randn(n, seed + 50 + k).to(dtype)
        params.append(p)
    return params


def alone(p, grads_and_hyper, bits):
    """The parameter stepped by itself, each step with its own options."""
    q = torch.nn.Parameter(p.clone())
    opt = FusedAdamW([q], state_bits=bits)
    for grad, hyper in grads_and_hyper:
        q.grad = grad
        opt.param_groups[0].update(hyper)
        opt.step()
    return q.detach()


@pytest.mark.parametrize("bits", [8, 32])
def test_groups_apply_their_own_options(bits):
    p = make([300, 400, 500])
    first = [t.detach().clone() for t in p]
    opt = FusedAdamW([{"params": p[:2], "lr": 1e-2}, {"params": p[2:], "weight_decay": 0.5, "eps": 1e-3}], lr=1e-3,
                     state_bits=bits)
    for _ in range(3):
        opt.step()
    options = [{k: v for k, v in opt.param_groups[i].items() if k != "params"} for i in (0, 0, 1)]
    assert options[0]["lr"] == 1e-2 and options[2]["weight_decay"] == 0.5
    for t, old, o in zip(p, first, options):
        assert torch.equal(t.detach(), alone(old, [(t.grad, o)] * 3, bits))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_parameter_taken_out_of_its_group_is_not_stepped(bits):
    p = make([300, 400, 500])
    opt = FusedAdamW(p, **HYPER, state_bits=bits)
    opt.step()
    kept = p[1].detach().clone()
    opt.param_groups[0]["params"] = [p[0], p[2]]
    opt.step()
    assert torch.equal(p[1], kept)
    assert not torch.equal(p[0], make([300, 400, 500])[0])


@pytest.mark.parametrize("bits", [8, 32])
def test_a_parameter_moved_to_another_group_keeps_its_state(bits):
    p = make([300, 400])
    first = p[1].detach().clone()
    opt = FusedAdamW([{"params": [p[0], p[1]], "lr": 1e-2}, {"params": make([64], 7), "lr": 1e-3}], state_bits=bits)
    opt.step()
    a, b = ({k: v for k, v in g.items() if k != "params"} for g in opt.param_groups)
    opt.param_groups[0]["params"] = [p[0]]
    opt.param_groups[1]["params"].append(p[1])
    opt.step()
    assert torch.equal(p[1].detach(), alone(first, [(p[1].grad, a), (p[1].grad, b)], bits))
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [2, 2, 2]


def test_a_group_that_is_removed_is_not_stepped_and_the_others_are():
    p = make([300, 400, 500])
    first = [t.detach().clone() for t in p]
    opt = FusedAdamW([{"params": [t], "lr": 10.0 ** -k} for k, t in enumerate(p)])
    opt.step()
    middle = p[0].detach().clone()
    options = [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups]
    del opt.param_groups[0]
    opt.step()
    assert torch.equal(p[0], middle)
    for k in (1, 2):
        assert torch.equal(p[k].detach(), alone(first[k], [(p[k].grad, options[k])] * 2, 32))
    assert len(opt.state_dict()["state"]) == 2


def test_a_parameter_replaced_by_another_is():
    p = make([300, 400])
    opt = FusedAdamW(p, **HYPER)
    opt.step()
    old, = make([400], 9)
    opt.param_groups[0]["params"][1] = old
    first, kept = old.detach().clone(), p[1].detach().clone()
    opt.step()
    assert torch.equal(p[1], kept) and torch.equal(old.detach(), alone(first, [(old.grad, HYPER)], 32))


def test_state_that_is_cleared_begins_anew():
    p = make([300, 400])
    opt = FusedAdamW(p, **HYPER)
    for _ in range(3):
        opt.step()
    opt.state.clear()
    first = [t.detach().clone() for t in p]
    opt.step()
    for t, old in zip(p, first):
        assert torch.equal(t.detach(), alone(old, [(t.grad, HYPER)], 32))
    del opt.state[p[0]]
    third = make([64], 5)
    third[0].grad = None
    opt.add_param_group({"params": third})
    first = p[0].detach().clone()
    third[0].grad = torch.ones(64, device="cuda")
    opt.step()
    assert torch.equal(p[0].detach(), alone(first, [(p[0].grad, HYPER)], 32))
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [1, 2, 1]


def test_looking_at_the_state_first_changes_nothing():
    p = make([300, 400])
    opt = FusedAdamW(p, **HYPER)
    assert not opt.state[p[0]]  # torch's state is a defaultdict: the entry is there now
    first = [t.detach().clone() for t in p]
    opt.step()
    assert not opt.state[torch.nn.Parameter(torch.zeros(1))]
    opt.step()
    for t, old in zip(p, first):
        assert torch.equal(t.detach(), alone(old, [(t.grad, HYPER)] * 2, 32))


def test_a_parameter_that_it_does_not_take_is_refused_in_a_changed_group():
    p = make([300])
    opt = FusedAdamW(p, **HYPER)
    opt.step()
    kept = p[0].detach().clone()
    for bad in (torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.float64))):
        bad.grad = torch.ones_like(bad)
        opt.param_groups[0]["params"].append(bad)
        with pytest.raises((RuntimeError, TypeError)):
            opt.step()
        opt.param_groups[0]["params"].pop()
    assert torch.equal(p[0], kept)


def test_a_parameter_given_twice_is_refused():
    """Its two steps would be one launch's, over the same values."""
    p, = make([300])
    with pytest.raises(ValueError):
        FusedAdamW([p, p])
    opt = FusedAdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [p]})
    opt.step()
    opt.param_groups[0]["params"].append(p)
    kept = p.detach().clone()
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(p, kept)
