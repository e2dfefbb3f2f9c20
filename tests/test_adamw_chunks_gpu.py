"""The 8-bit AdamW step where a thread block has several chunks, one after the
other through its ring of copies: from some 7 million elements on.  State to the
bit, parameters against the formula (tolerances: test_adamw_gpu.py)."""
import pytest
import torch

from mlp_megakernel_b200 import FusedAdamW

from .test_adamw_gpu import HYPER, U, W, formula, quantize, randn, values

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def with_gradient(n, dtype, g_dtype, offset, seed):
    p = torch.nn.Parameter(randn(n + offset, seed, 0.5).to(dtype)[offset:])
    if g_dtype != dtype:
        p.grad_dtype = g_dtype
    p.grad = torch.zeros(n + offset, device="cuda", dtype=g_dtype)[offset:]
    return p


@pytest.mark.parametrize("dtype,g_dtype,master", [(F32, F32, False), (F16, F16, False), (BF16, BF16, False),
                                                  (BF16, BF16, True), (F16, F32, False), (F16, F32, True)])
@pytest.mark.parametrize("sizes,offset", [
    ([8_000_001, 4097, 300_001, 7], 0),  # 2 chunks a thread block
    ([5_000_000, 6_500_009], 1),         # 3, none of them aligned
    ([30_000_003, 2048, 2049], 0),       # 8
    ([60_000_000], 0),                   # 16
])
def test_several_chunks_a_block(dtype, g_dtype, master, sizes, offset):
    try:
        params = [with_gradient(n, dtype, g_dtype, offset, k) for k, n in enumerate(sizes)]
    except (AttributeError, RuntimeError):
        pytest.skip("this torch keeps gradients in the parameter's type")
    opt = FusedAdamW(params, **HYPER, master_weights=master, state_bits=8)
    b1, b2 = HYPER["betas"]
    before = [(p.detach().float().clone(), torch.zeros_like(p, dtype=F32), torch.zeros_like(p, dtype=F32)) for p in params]
    for t in (1, 2, 3):
        for k, p in enumerate(params):
            p.grad.copy_(randn(p.numel(), 100 * t + k, 0.1))
            p.grad[: p.numel() // 3] *= 1e-3
        opt.step()
        for k, p in enumerate(params):
            s, (old, m, r), g = opt.state[p], before[k], p.grad.float()
            got = s["master_param"] if master else p.detach()
            for a in range(0, p.numel(), 1 << 24):  # in parts, for the memory of the 64-bit formula
                e = slice(a, a + (1 << 24))
                new, *_, room = formula(old[e].double(), g[e].double(), m[e].double(), r[e].double().square(), t, **HYPER)
                u = W if master else U[dtype]
                assert ((got[e].double() - new).abs() <= u * new.abs() + W * room + 2.0 ** -25).all()
            m = m * b1 + g * (1 - b1)
            v = (r * r) * b2 + (g * g) * (1 - b2)
            (mq, m_scale), (rq, r_scale) = quantize(m, False), quantize(v.sqrt(), True)
            assert torch.equal(s["exp_avg"].float(), mq.float()) and torch.equal(s["exp_avg_scale"], m_scale)
            assert torch.equal(s["exp_avg_rms"].float(), rq.float()) and torch.equal(s["exp_avg_rms_scale"], r_scale)
            before[k] = got.float().clone(), values(mq, m_scale), values(rq, r_scale)
