"""A value before the activation that is NaN: so are the output and every gradient that depends on it, whatever the
activation; the others are what they are without it."""
import pytest
import torch

from mlp_megakernel_b200 import _lib, feedforward as ff

pytestmark = pytest.mark.gpu
ops = torch.ops.mlpk
ACTS = [a for a in ff.ACTIVATIONS if a is not None]


@pytest.fixture(autouse=True)
def status():
    yield
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def randn(*shape, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(*shape, device="cuda", generator=g)).to(dtype)


@pytest.mark.parametrize("rows", [5, 150, 700])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_nan_before_the_activation(rows, act, dtype):
    code = ff.ACTIVATIONS[act]
    x, w, wu = (randn(*s, seed=k, dtype=dtype, scale=0.3) for k, s in enumerate(((rows, 72), (72, 136), (72, 136))))
    wd, go, gd = (randn(*s, seed=k, dtype=dtype) for k, s in enumerate(((136, 40), (rows, 136), (rows, 40)), 3))
    for keep in (1, 2):
        # linear: z[2, 11], or in 8 bits its group of row 2
        out, z, *s = ops.linear(x, w, None, None, code, keep)
        s = s[0] if s else None
        bad_z, bad_s = z.clone(), None if s is None else s.clone()
        if keep == 1:
            bad_z[2, 11] = float("nan")
        else:
            bad_s[2, 0] = float("nan")
        want = ops.linear_bwd(go, x, None, w, z, s, code, dtype, True, True, True)
        got = ops.linear_bwd(go, x, None, w, bad_z, bad_s, code, dtype, True, True, True)
        rest = [r for r in range(rows) if r != 2]
        assert got[0][2].isnan().all() and torch.equal(got[0][rest], want[0][rest])
        lost = torch.zeros(136, dtype=torch.bool, device="cuda")
        lost[11 if keep == 1 else slice(0, 128)] = True
        for a, b in zip(got[1:], want[1:]):
            assert a[..., lost].isnan().all() and torch.equal(a[..., ~lost], b[..., ~lost])
        # gate
        _, *k = ops.gated_mlp(x, w, wu, wd, None, code, keep)
        g, gs, u, us = k if keep == 2 else (k[0], None, k[1], None)
        bad_g, bad_s = g.clone(), None if gs is None else gs.clone()
        if keep == 1:
            bad_g[2, 11] = float("nan")
        else:
            bad_s[2, 0] = float("nan")
        want = ops.gated_mlp_bwd(gd, x, None, w, wu, wd, g, gs, u, us, code, True, True, True)
        got = ops.gated_mlp_bwd(gd, x, None, w, wu, wd, bad_g, bad_s, u, us, code, True, True, True)
        assert got[0][2].isnan().all() and torch.equal(got[0][rest], want[0][rest])
        for a, b in ((got[1], want[1]), (got[2], want[2]), (got[3].t(), want[3].t())):
            assert a[..., lost].isnan().all() and torch.equal(a[..., ~lost], b[..., ~lost])
