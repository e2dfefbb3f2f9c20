"""What FusedAdamW refuses, loads and calls before there is any state (no GPU
needed)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlp_megakernel_b200 as m


@pytest.fixture
def opt():
    with FakeTensorMode():
        yield m.FusedAdamW([torch.nn.Parameter(torch.empty(8, device="cuda"))], lr=1e-3)


@pytest.mark.parametrize("change", [dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(0.9, 1.0)), dict(eps=-1.0)])
def test_a_refused_load_keeps_the_options(opt, change):
    saved = opt.state_dict()
    saved["param_groups"][0].update(change)
    with pytest.raises(ValueError):
        opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == 1e-3 and opt.param_groups[0]["betas"] == (0.9, 0.999)
    assert opt.param_groups[0]["eps"] == 1e-8


def test_hooks_are_called(opt):
    said = []
    opt.register_state_dict_pre_hook(lambda o: said.append("pre"))
    opt.register_state_dict_post_hook(lambda o, d: said.append("post") or {**d, "more": 1})
    opt.register_load_state_dict_pre_hook(lambda o, d: said.append("load") or
                                          {**d, "param_groups": [{**g, "lr": 0.5} for g in d["param_groups"]]})
    opt.register_load_state_dict_post_hook(lambda o: said.append("loaded"))
    saved = opt.state_dict()
    assert saved["more"] == 1
    opt.load_state_dict(saved)
    assert said == ["pre", "post", "load", "loaded"] and opt.param_groups[0]["lr"] == 0.5
    assert saved["param_groups"][0]["lr"] == 1e-3  # the caller's dict is not changed


def test_duplicates_are_refused(opt):
    p = opt.param_groups[0]["params"][0]
    with pytest.raises(ValueError):
        m.FusedAdamW([p, p])
