"""Loads of FusedAdamW's state: one that is refused changes nothing, and a tensor
lr may come from another device."""
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


def tensors_of(opt):
    return [t.clone() for flat in opt.flat_state() for t in flat.values()]


@pytest.mark.parametrize("change", [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.5),
                                    dict(lr=torch.tensor(1e-3, dtype=torch.float64)),
                                    dict(lr=torch.tensor([1e-3, 1e-3]))])
@pytest.mark.parametrize("group", [0, 1])
def test_a_refused_load_changes_nothing(change, group):
    p = make([300, 1, 5000], dtype=torch.float16)
    opt = FusedAdamW([{"params": p[:2]}, {"params": p[2:], "lr": 1e-2}], **HYPER, master_weights=True)
    for _ in range(2):
        opt.step()
    saved = opt.state_dict()
    saved["param_groups"][group].update(change)
    before, options = tensors_of(opt), [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups]
    buffers = [t.data_ptr() for flat in opt.flat_state() for t in flat.values()]
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    assert [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups] == options
    assert [t.data_ptr() for flat in opt.flat_state() for t in flat.values()] == buffers
    assert all(torch.equal(a, b) for a, b in zip(tensors_of(opt), before))
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [2, 2, 2]
    opt.step()
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [3, 3, 3]


def test_a_tensor_lr_read_to_the_host_is_taken():
    p, q = make([700]), make([700])
    a = FusedAdamW(p, lr=torch.tensor(3e-3, device="cuda"))
    a.step()
    saved = a.state_dict()
    saved = {"state": {k: {n: v.cpu() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
                       for k, s in saved["state"].items()},
             "param_groups": [{**g, "lr": g["lr"].cpu()} for g in saved["param_groups"]]}
    with torch.no_grad():
        q[0].copy_(p[0])
    for start in (1.0, torch.tensor(1.0, device="cuda")):
        b = FusedAdamW([q[0]], lr=start)
        b.load_state_dict(saved)
        assert b.param_groups[0]["lr"].device == p[0].device and b.param_groups[0]["lr"].item() == a.param_groups[0]["lr"].item()
    a.step()
    b.step()
    assert torch.equal(p[0], q[0])


@pytest.mark.parametrize("step", [-1, None, float("nan")])
def test_a_refused_step_count_changes_nothing(step):
    p = make([40, 300])
    opt = FusedAdamW(p, **HYPER)
    opt.step()
    saved, before = opt.state_dict(), tensors_of(opt)
    saved["state"][1]["step"] = step
    with pytest.raises((ValueError, TypeError)):
        opt.load_state_dict(saved)
    assert all(torch.equal(a, b) for a, b in zip(tensors_of(opt), before))
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [1, 1]


@pytest.mark.parametrize("bits", [8, 32])
def test_its_own_state_loaded_again(bits):
    """The tensors of the dict are the optimizer's own buffers."""
    p, q = make([300, 1, 5000], dtype=torch.float16), make([300, 1, 5000], dtype=torch.float16)
    a, b = (FusedAdamW(t, **HYPER, state_bits=bits, master_weights=True) for t in (p, q))
    for opt in (a, b):
        opt.step()
    a.load_state_dict(a.state_dict())
    for opt in (a, b):
        opt.step()
    assert all(torch.equal(x, y) for x, y in zip(p, q))


def test_hooks_of_state_dict_and_load():
    """Called as torch's optimizers call them; a result replaces the dict."""
    p = make([40])
    opt = FusedAdamW(p, **HYPER)
    opt.step()
    said = []
    opt.register_state_dict_pre_hook(lambda o: said.append(("pre", o is opt)))
    opt.register_state_dict_post_hook(lambda o, d: {**d, "more": len(d["state"])})
    opt.register_load_state_dict_pre_hook(lambda o, d: said.append(("load", "more" in d)) or
                                          {k: v for k, v in d.items() if k != "more"})
    opt.register_load_state_dict_post_hook(lambda o: said.append(("loaded", o.state_dict()["state"][0]["step"])))
    saved = opt.state_dict()
    assert saved["more"] == 1 and saved["state"][0]["step"] == 1
    opt.step()
    opt.load_state_dict(saved)
    assert said == [("pre", True), ("load", True), ("pre", True), ("loaded", 1)]
    opt.register_load_state_dict_pre_hook(lambda o, d: d["param_groups"][0].update(lr=-1.0))
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == HYPER["lr"]
