"""The AdamW step against its formula in 64 bits, and its 8-bit state against
the same operations in fp32, one at a time.

Tolerances, w = 2^-24 being fp32's unit roundoff and u the parameter type's.
m: two products and a sum: 3 w (|b1 m| + |(1-b1) g|), and w more for each of the
constants in fp32: 4 w of that sum.  v: 6 w of its (positive) terms.  p: the
update's relative error is that of m (against |b1 m| + |(1-b1) g|), half of v's,
and at most 16 w for the two corrections, the root, the sum and the quotients;
p's own product and sum add 3 w |p|.
"""
import pytest
import torch

from mlp_megakernel_b200 import FusedAdamW, FusedMLPSoftplus

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
W = 2.0 ** -24
SIZES = [1, 7, 8, 255, 256, 257, 4095, 4096, 4097, 20001]
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def randn(n, seed, scale=1.0):
    return scale * torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def make(sizes, dtype, g_dtype=None, offset=0, seed=0):
    """Parameters (each `offset` elements into an allocation) with gradients."""
    params = []
    for k, n in enumerate(sizes):
        p = torch.nn.Parameter(randn(n + offset, seed + k, 0.5).to(dtype)[offset:])
        if g_dtype in (None, dtype):
            p.grad = randn(n + offset, seed + 100 + k, 0.1).to(dtype)[offset:]
        else:
            p.grad_dtype = g_dtype
            p.grad = randn(n + offset, seed + 100 + k, 0.1).to(g_dtype)[offset:]
        params.append(p)
    return params


def formula(p, g, m, v, t, lr, betas, eps, weight_decay):
    """(p, m, v) after step t in 64 bits, and what the tolerances are shares of."""
    b1, b2 = betas
    m_room = (b1 * m).abs() + ((1 - b1) * g).abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    denom = (v / (1 - b2 ** t)).sqrt() + eps
    new = p * (1 - lr * weight_decay) - lr / (1 - b1 ** t) * m / denom
    p_room = 3 * p.abs() + lr / (1 - b1 ** t) * (4 * m_room + 20 * m.abs()) / denom
    return new, m, v, m_room, p_room


@pytest.mark.parametrize("dtype,g_dtype,master", [
    (torch.float32, None, False), (torch.float16, None, False), (torch.bfloat16, None, False),
    (torch.float16, None, True), (torch.bfloat16, None, True)])
@pytest.mark.parametrize("offset", [0, 1])
def test_steps_in_32_bits(dtype, g_dtype, master, offset):
    params = make(SIZES, dtype, g_dtype, offset)
    opt = FusedAdamW(params, **HYPER, master_weights=master)
    values = [p.detach().double() for p in params]
    ms, vs = ([torch.zeros_like(v) for v in values] for _ in range(2))
    for t in range(1, 4):
        for k, p in enumerate(params):
            p.grad.copy_(randn(p.numel(), 1000 * t + k, 0.1))
            if t == 2:
                p.grad[: p.numel() // 2] = 0
        opt.step()
        for k, p in enumerate(params):
            s = opt.state[p]
            new, m, v, m_room, p_room = formula(values[k], p.grad.double(), ms[k], vs[k], t, **HYPER)
            assert ((s["exp_avg"].double() - m).abs() <= 4 * W * m_room + 1e-45).all()
            assert ((s["exp_avg_sq"].double() - v).abs() <= 6 * W * v + 1e-45).all()
            got = s["master_param"] if master else p.detach()
            u = W if master else U[dtype]
            assert ((got.double() - new).abs() <= u * new.abs() + W * p_room + 2.0 ** -25).all()
            if master:
                assert torch.equal(p.detach(), got.to(dtype))
            values[k], ms[k], vs[k] = got.double(), s["exp_avg"].double(), s["exp_avg_sq"].double()
    assert all(s["step"] == 3 for s in opt.state_dict()["state"].values())


def test_gradients_in_fp32_beside_16_bits():
    """A 16-bit parameter whose gradient is fp32: through the C ABI's g_dtype."""
    p = torch.nn.Parameter(randn(1000, 1).half())
    q = torch.nn.Parameter(randn(500, 2).half())
    try:
        p.grad_dtype = torch.float32
        p.grad = randn(1000, 3, 0.1)
    except (AttributeError, RuntimeError):
        pytest.skip("this torch keeps gradients in the parameter's type")
    q.grad = randn(500, 4, 0.1).half()
    before = [t.detach().double() for t in (p, q)]
    opt = FusedAdamW([p, q], **HYPER)
    opt.step()
    for t, old in zip((p, q), before):
        new, *_, room = formula(old, t.grad.double(), old * 0, old * 0, 1, **HYPER)
        assert ((t.detach().double() - new).abs() <= U[torch.float16] * new.abs() + W * room + 2.0 ** -25).all()


def quantize(v, least):
    """Blocks of 256 in fp32, operation by operation as the kernel's comment says."""
    n = v.numel()
    b = torch.nn.functional.pad(v, (0, -n % 256)).view(-1, 256)
    scale = b.abs().amax(1) * torch.tensor(1.0 / 448.0, device="cuda")
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, 0.0, scale)
    q = b * torch.where(scale > 0, 1.0 / scale, 0.0)[:, None]
    if least:
        q = torch.where((b > 0) & (scale > 0)[:, None], q.clamp(min=2.0 ** -9), q)
    return q.clamp(-448, 448).to(torch.float8_e4m3fn).view(-1)[:n], scale


def values(q, scale):
    n = q.numel()
    return (torch.nn.functional.pad(q.float(), (0, -n % 256)).view(-1, 256) * scale[:, None]).view(-1)[:n]


@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.float16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("offset", [0, 1])
def test_steps_in_8_bits(dtype, master, offset):
    """The state after each step is the fp32 operations' to the bit; the
    parameters follow the formula from the state's values before the step."""
    params = make(SIZES, dtype, None, offset)
    opt = FusedAdamW(params, **HYPER, master_weights=master, state_bits=8)
    b1, b2 = HYPER["betas"]
    olds = [p.detach().double() for p in params]
    state = [(torch.zeros_like(p, dtype=torch.float32),) * 2 for p in params]
    for t in range(1, 5):
        for k, p in enumerate(params):
            p.grad.copy_(randn(p.numel(), 1000 * t + k, 0.1 * 10.0 ** -(k % 4)))
            p.grad[: p.numel() // 3] *= 1e-3
            if t > 2:
                p.grad[: p.numel() // 4] = 0
        opt.step()
        for k, p in enumerate(params):
            s, (m, r) = opt.state[p], state[k]
            g = p.grad.float()
            new, *_, room = formula(olds[k], g.double(), m.double(), r.double().square(), t, **HYPER)
            m = m * b1 + g * (1 - b1)
            v = (r * r) * b2 + (g * g) * (1 - b2)
            (mq, m_scale), (rq, r_scale) = quantize(m, False), quantize(v.sqrt(), True)
            assert torch.equal(s["exp_avg"].float(), mq.float()) and torch.equal(s["exp_avg_scale"], m_scale)
            assert torch.equal(s["exp_avg_rms"].float(), rq.float()) and torch.equal(s["exp_avg_rms_scale"], r_scale)
            assert (rq.float()[v > 0] > 0).all()
            state[k] = values(mq, m_scale), values(rq, r_scale)
            got = s["master_param"] if master else p.detach()
            u = W if master else U[dtype]
            assert ((got.double() - new).abs() <= u * new.abs() + W * room + 2.0 ** -25).all()
            olds[k] = got.double()


def test_state_in_8_bits_at_its_ends():
    """Zero gradients, gradients whose squares and scales underflow, and one
    that is not finite: its block of 256 is NaN, the others are not."""
    p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
    p.grad = torch.zeros(1024, device="cuda")
    p.grad[256:512] = 1e-38
    p.grad[512:768] = 1e-22
    p.grad[513] = 1e-3
    p.grad[800] = float("inf")
    opt = FusedAdamW([p], lr=1e-2, weight_decay=0.0, state_bits=8)
    for _ in range(3):
        opt.step()
    assert torch.equal(p.detach()[:256], torch.ones(256, device="cuda"))
    assert p.detach()[256:768].isfinite().all() and (p.detach()[256:768] - 1).abs().max().item() < 0.1
    assert not p.detach()[768:][torch.arange(256, device="cuda") == 32].isfinite().any()
    s = opt.state[p]
    assert s["exp_avg_scale"][:3].isfinite().all() and not s["exp_avg_scale"][3].isfinite()
    assert not s["exp_avg"].float()[:256].any()


def test_many_tensors_of_mixed_types():
    """More tensors than one launch's table, of all types in one group, some of
    no elements: the same as tensor by tensor."""
    sizes = [(i * 37) % 700 for i in range(1700)]
    kinds = [torch.float32, torch.float16, torch.bfloat16]
    a = [torch.nn.Parameter(randn(n, i).to(kinds[i % 3])) for i, n in enumerate(sizes)]
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    together = FusedAdamW(a, **HYPER, state_bits=8)
    apart = [FusedAdamW([p], **HYPER, state_bits=8) for p in b]
    for t in range(2):
        for i, (p, q) in enumerate(zip(a, b)):
            p.grad = q.grad = randn(p.numel(), 5000 + i + t, 0.1).to(p.dtype)
        together.step()
        for opt in apart:
            opt.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_parameters_without_gradient_and_groups():
    p = make([300, 400, 500], torch.float32)
    opt = FusedAdamW([{"params": p[:2], "lr": 1e-2}, {"params": p[2:], "weight_decay": 0.5}], lr=1e-3)
    opt.step()
    grad, p[1].grad = p[1].grad, None
    before = p[1].detach().clone()
    opt.step()
    assert torch.equal(p[1], before)
    p[1].grad = grad
    opt.step()
    steps = [s["step"] for s in opt.state_dict()["state"].values()]
    assert steps == [3, 2, 3]
    late = make([64], torch.float32, seed=9)
    late[0].grad = None
    opt.add_param_group({"params": late})
    opt.step()
    late[0].grad = torch.ones(64, device="cuda")
    opt.step()
    assert [s["step"] for s in opt.state_dict()["state"].values()] == [5, 4, 5, 1]
    torch_p = [torch.nn.Parameter(t.detach().clone()) for t in p]
    assert len(torch_p) == 3


def test_against_torch():
    """Ten steps beside torch.optim.AdamW in 64 bits; each step may differ by the
    tolerance above, so ten of them by ten times its largest value (and the
    update of the next steps by as much again)."""
    p = make([1000, 4097], torch.float32)
    q = [torch.nn.Parameter(t.detach().double()) for t in p]
    hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    a, b = FusedAdamW(p, **hyper, maximize=True), torch.optim.AdamW(q, **hyper, maximize=True)
    for t in range(10):
        for k, (x, y) in enumerate(zip(p, q)):
            x.grad = randn(x.numel(), 77 * t + k)
            y.grad = x.grad.double()
        a.step()
        b.step()
    for x, y in zip(p, q):
        assert (x.double() - y).abs().max().item() <= 10 * W * (3 * y.abs().max().item() + 100 * 1e-2)


@pytest.mark.parametrize("bits", [8, 32])
def test_betas_of_zero(bits):
    """m = g and r = |g|: the step is lr * sign(g), as far as |g| is above eps."""
    p = torch.nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad = randn(300, 1).clamp(min=0.1) * torch.where(randn(300, 2) > 0, 1.0, -1.0)
    opt = FusedAdamW([p], lr=0.5, betas=(0.0, 0.0), eps=1e-12, weight_decay=0.0, state_bits=bits)
    opt.step()
    assert ((p.detach() + 0.5 * p.grad.sign()).abs() <= 0.5 * 20 * W).all()


def test_strides_and_orders():
    """A transposed parameter, a gradient of another order, and one that is a
    slice: elements meet their own gradient."""
    w = torch.nn.Parameter(randn(60 * 40, 1).view(60, 40).t())
    flat = torch.nn.Parameter(w.detach().contiguous())
    g = randn(2400, 2, 0.1).view(40, 60)
    a, b = FusedAdamW([w], **HYPER), FusedAdamW([flat], **HYPER)
    for grad in (g, g.t().contiguous().t(), torch.cat([g, g], 1)[:, :60]):
        w.grad, flat.grad = grad, g
        a.step()
        b.step()
    assert torch.equal(w.detach(), flat.detach())
    assert torch.equal(a.state[w]["exp_avg"], b.state[flat]["exp_avg"])


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("master", [False, True])
def test_state_dict(bits, master):
    def fresh():
        p = make([300, 1, 5000], torch.float16)
        return p, FusedAdamW(p, **HYPER, state_bits=bits, master_weights=master)

    p, a = fresh()
    for _ in range(3):
        a.step()
    q, b = fresh()
    with torch.no_grad():
        for x, y in zip(p, q):
            y.copy_(x)
    saved = a.state_dict()
    b.load_state_dict(saved)
    for opt in (a, b):
        opt.param_groups[0]["lr"] = 1e-3
        opt.step()
        opt.step()
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    assert [s["step"] for s in b.state_dict()["state"].values()] == [5, 5, 5]
    for x, y in zip(a.flat_state(), b.flat_state()):
        assert x.keys() == y.keys() and all(torch.equal(x[k].float(), y[k].float()) for k in x)
    wrong = {"state": {0: {"step": 1, "exp_avg": p[0]}}, "param_groups": saved["param_groups"]}
    with pytest.raises(ValueError):
        b.load_state_dict(wrong)
    with pytest.raises(ValueError):
        FusedAdamW(make([3], torch.float16)[:1]).load_state_dict(saved)


def test_grad_scale_found_inf_and_scaler():
    p, q = make([5000], torch.float32)[0], make([5000], torch.float32)[0]
    a, b = FusedAdamW([p], **HYPER), FusedAdamW([q], **HYPER)
    p.grad *= 1024
    one, zero = torch.ones((), device="cuda"), torch.zeros((), device="cuda")
    a.step(grad_scale=one * 1024, found_inf=zero)
    b.step()
    assert torch.equal(p, q)  # a power of two
    before = [t.clone() for t in (p.detach(), *a.flat_state()[0].values())]
    a.step(grad_scale=one * 1024, found_inf=one)
    assert all(torch.equal(x, y) for x, y in zip(before, (p.detach(), *a.flat_state()[0].values())))
    assert a.state_dict()["state"][0]["step"] == 1
    scaler = torch.amp.GradScaler("cuda", init_scale=256.0)
    model = FusedMLPSoftplus(D=32, H=64, out_features=16, num_layers=5).cuda()
    opt = FusedAdamW(model.parameters(), lr=1e-3)
    x = torch.randn(300, 32, device="cuda")
    for k in range(3):
        opt.zero_grad()
        loss = model(x).float().square().mean()
        scaler.scale(loss).backward()
        if k == 1:
            model.w1.grad[0, 0] = float("nan")
        scaler.step(opt)
        scaler.update()
    assert all(s["step"] == 2 for s in opt.state_dict()["state"].values())
    assert all(w.isfinite().all() for w in model.parameters())


def test_lr_tensor_and_graph():
    """A captured step replays with new gradients, a new lr, and counts."""
    p, q = make([3000, 17], torch.float32), make([3000, 17], torch.float32)
    lr = torch.tensor(1e-2, device="cuda")
    a, b = FusedAdamW(p, lr=lr), FusedAdamW(q, lr=1e-2)
    a.step()
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for t in range(3):
        lr.fill_(1e-2 / (t + 1))
        b.param_groups[0]["lr"] = float(lr)
        for x, y in zip(p, q):
            y.grad = randn(x.numel(), t, 0.3)
            x.grad.copy_(y.grad)
        graph.replay()
        b.step()
    for x, y in zip(p, q):
        assert torch.equal(x, y)
    assert [s["step"] for s in a.state_dict()["state"].values()] == [4, 4]


def test_another_stream():
    p, q = make([9000], torch.float32)[0], make([9000], torch.float32)[0]
    a, b = FusedAdamW([p], **HYPER), FusedAdamW([q], **HYPER)
    a.step()
    b.step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        p.grad = p.detach() * 2
        a.step()
    torch.cuda.current_stream().wait_stream(s)
    q.grad = q.detach() * 2
    b.step()
    assert torch.equal(p, q)


def test_a_parameter_of_the_graph_is_known_to_have_changed():
    w = torch.nn.Parameter(randn(10, 1))
    w.grad = torch.ones(10, device="cuda")
    loss = (w * w).sum()
    FusedAdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_closure_and_scheduler():
    p = make([100], torch.float32)
    opt = FusedAdamW(p, lr=0.1)
    schedule = torch.optim.lr_scheduler.StepLR(opt, 1, 0.1)
    calls = []
    assert opt.step(lambda: calls.append(torch.is_grad_enabled()) or 7) == 7 and calls == [True]
    schedule.step()
    assert abs(opt.param_groups[0]["lr"] - 0.01) < 1e-12


def test_more_than_32_bits_of_elements():
    """A tensor of more than 2^31 elements: its last ones are stepped."""
    n = 2 ** 31 + 4500
    p = torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    opt = FusedAdamW([p], lr=0.25, weight_decay=0.0, eps=0.0, state_bits=8)
    opt.step()
    tail = p.detach()[-5000:].float()
    assert (tail == -0.25).all() and (p.detach()[:1000].float() == -0.25).all()
