"""What is measured of the block operators: the RMS norm with the residual's addition, the rows sorted by expert and
back, and the AdamW step over many tensors.

Each operator has a plain form in elementary torch operations (fp32 throughout, one rounding at the end) next to the
call of the framework's own kernels, and a statement of its definition in 64 bits (``exact``).
"""
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6
E4M3_MAX = 448.0
E4M3_TINY = 2.0 ** -9  # smallest positive value of the 8-bit type
BLOCK = 256  # elements that share a scale of the 8-bit optimizer state
LR, BETA1, BETA2, ADAM_EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 0.01
STEP = 1000  # steps taken before the measured one


def listed():
    return [
        # one token's row at a decoding step: latency
        dict(name="norm_one_row", op="norm", rows=1, width=4096, dtype="bf16", residual=True, train=False),
        # a training batch's residual stream
        dict(name="norm_train", op="norm", rows=16384, width=4096, dtype="bf16", residual=True, train=True),
        # the fused MLP's own rows: 128 wide, a quarter of a million of them
        dict(name="norm_train_narrow", op="norm", rows=262144, width=128, dtype="f16", residual=True, train=True),
        # rows for a projection in 8 bits, a scale for every 128 columns
        dict(name="norm_fp8", op="fp8", rows=8192, width=5120, dtype="bf16", residual=True, group=128),
        # rows that no vector load divides, a scale a row
        dict(name="norm_fp8_odd", op="fp8", rows=5003, width=1999, dtype="f16", residual=False, group=0),
        # a small decoding batch through eight experts
        dict(name="experts_decode", op="experts", tokens=8, top=2, experts=8, width=256, dtype="f16", ids="i64", drop=0.0, train=False),
        # a long prompt through many experts
        dict(name="experts_prompt", op="experts", tokens=32768, top=8, experts=64, width=2048, dtype="bf16", ids="i64", drop=0.0, train=False),
        # a training batch of the fused MLP's widest rows, some slots over their expert's capacity
        dict(name="experts_train", op="experts", tokens=131072, top=2, experts=16, width=256, dtype="f16", ids="i64", drop=0.05, train=True),
        # rows that no vector load divides, in 32 bits
        dict(name="experts_train_odd", op="experts", tokens=9973, top=3, experts=37, width=517, dtype="f32", ids="i32", drop=0.1, train=True),
        # the 5-layer 32-64-64-64-64-16 network: latency
        dict(name="adamw_small", op="adamw", shapes="32x64,64x64*3,64x16", dtype="f32", bits=32, master=False),
        # matrices and vectors of a larger model in 16 bits, the state in 8
        dict(name="adamw_8bit", op="adamw", shapes="4096x4096*12,4096x1024*8,4096*24", dtype="bf16", bits=8, master=False),
        # many tensors of odd sizes in 16 bits, their 32-bit copies and state beside them
        dict(name="adamw_many", op="adamw", shapes="1000x777*120,333x1001*60,1001*180", dtype="f16", bits=32, master=True),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["norm", "norm", "fp8", "experts", "experts", "adamw", "adamw"])
    if op in ("norm", "fp8"):
        width = _log(rng, 24, 16384)
        if rng.random() < 0.7:
            width = -(-width // 8) * 8
        rows = _log(rng, 1, min(262144, (1 << 26) // width))
        case = dict(op=op, rows=rows, width=width, dtype=rng.choice(["f16", "bf16", "f32"]), residual=rng.random() < 0.7)
        return {**case, "group": rng.choice([0, 128])} if op == "fp8" else {**case, "train": rng.random() < 0.6}
    if op == "experts":
        width = _log(rng, 24, 8192)
        if rng.random() < 0.7:
            width = -(-width // 8) * 8
        experts = _log(rng, 2, 384)
        top = min(experts, rng.randint(1, 8))
        tokens = _log(rng, 1, min(262144, (1 << 27) // (width * top)))
        return dict(op=op, tokens=tokens, top=top, experts=experts, width=width, dtype=rng.choice(["f16", "bf16", "f32"]),
                    ids=rng.choice(["i64", "i32"]), drop=rng.choice([0.0, 0.0, 0.05, 0.5]), train=rng.random() < 0.6)
    a, b, n, m = _log(rng, 8, 2048), _log(rng, 8, 2048), _log(rng, 1, 24), _log(rng, 1, 60)
    dtype, bits = rng.choice(["f16", "bf16", "f32"]), rng.choice([8, 32])
    return dict(op=op, shapes="%dx%d*%d,%d*%d" % (a, b, n, b, m), dtype=dtype, bits=bits, master=dtype != "f32" and bits == 32 and rng.random() < 0.5)


def _numels(shapes):
    """The sizes of the tensors that a text such as "64x64*3,64" names."""
    found = []
    for part in shapes.split(","):
        shape, _, count = part.partition("*")
        n = 1
        for d in shape.split("x"):
            n *= int(d)
        found += [n] * int(count or 1)
    return found


def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, scale, generator=g)

    return g, normal


def prepare(case, seed):
    g, normal = _random(seed)
    dt = DTYPES[case["dtype"]] if "dtype" in case else None
    if case["op"] in ("norm", "fp8"):
        rows, width, train = case["rows"], case["width"], case.get("train", False)
        s = {"case": case, "x": normal(rows, width, dtype=dt), "w": (1 + normal(width, scale=0.1)).to(dt),
             "r": normal(rows, width, dtype=dt, scale=2.0) if case["residual"] else None}
        if train:
            s["gy"] = normal(rows, width, dtype=dt, scale=0.1)
            s["gh"] = normal(rows, width, dtype=dt, scale=0.1) if case["residual"] else None
            for k in ("x", "w", "r"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
        return s
    if case["op"] == "experts":
        T, K, E, D = case["tokens"], case["top"], case["experts"], case["width"]
        # a router's choice: some experts are liked better than others
        scores, ids = (normal(T, E) + normal(E)).topk(K, dim=1)
        w = torch.softmax(scores, dim=1)
        if case["drop"]:
            ids = torch.where(torch.rand(T, K, device="cuda", generator=g) < case["drop"], -1, ids)
        s = {"case": case, "ids": ids.to(torch.int64 if case["ids"] == "i64" else torch.int32).contiguous(), "w": w.contiguous(),
             "x": normal(T, D, dtype=dt), "y": normal(T * K, D, dtype=dt)}
        if case["train"]:
            s["gxs"], s["gout"] = normal(T * K, D, dtype=dt, scale=0.1), normal(T, D, dtype=dt, scale=0.1)
            for k in ("x", "y", "w"):
                s[k].requires_grad_(True)
        return s
    # The parameters and their gradients, each tensor at a multiple of BLOCK elements of one buffer, and the state
    # of a run that has taken STEP steps.
    numels = _numels(case["shapes"])
    first, total = [], 0
    for n in numels:
        first.append(total)
        total += -(-n // BLOCK) * BLOCK
    master, grad = normal(total, scale=0.02), normal(total, dtype=dt, scale=1e-2)
    m, r = normal(total, scale=3e-3), normal(total, scale=1e-2).abs_()
    for off, n, nxt in zip(first, numels, first[1:] + [total]):
        for t in (master, grad, m, r):
            t[off + n:nxt] = 0
    p = master.to(dt)
    s = {"case": case, "p": p, "g": grad, "t": STEP}
    if case["master"]:
        s["master"] = master
    if case["bits"] == 8:
        (s["m"], s["ms"]), (s["r"], s["rs"]) = _quantize(m, 0.0), _quantize(r, E4M3_TINY)
    else:
        s["m"], s["v"] = m, r.square()
    if own:
        from mlp_megakernel_b200 import FusedAdamW

        params = []
        for off, n in zip(first, numels):
            q = torch.nn.Parameter(p[off:off + n])
            q.grad = grad[off:off + n]
            params.append(q)
        opt = FusedAdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"],
                         master_weights=case["master"])
        state = {}
        for i, (off, n) in enumerate(zip(first, numels)):
            b, e = off // BLOCK, off // BLOCK - (-n // BLOCK)
            state[i] = {"step": STEP, "exp_avg": s["m"][off:off + n]}
            if case["bits"] == 8:
                state[i].update(exp_avg_scale=s["ms"][b:e], exp_avg_rms=s["r"][off:off + n], exp_avg_rms_scale=s["rs"][b:e])
            else:
                state[i].update(exp_avg_sq=s["v"][off:off + n])
            if case["master"]:
                state[i].update(master_param=master[off:off + n])
        opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
        s = {"case": case, "p": p, "opt": opt}
    return s


def _quantize(v, least):
    """(8-bit values, scale of each BLOCK): the largest of a block becomes 448; what is above 0 becomes `least` at least."""
    b = v.view(-1, BLOCK)
    scale = b.abs().amax(dim=1) * (1 / E4M3_MAX)
    q = b * torch.where(scale > 0, 1 / scale, 0.0)[:, None]
    if least:
        q = torch.where(b > 0, q.clamp(min=least), q)
    return q.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(-1), scale


# ---------------------------------------------------------------- plain forms
def _norm_plain(s):
    c = s["case"]
    h = s["x"].float() + s["r"].float() if c["residual"] else s["x"].float()
    rstd = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS)
    return h, rstd, h * rstd * s["w"].float()


def _run_norm(s):
    c = s["case"]
    if own:
        from mlp_megakernel_b200 import fused_rms_norm

        if not c["train"]:
            got = fused_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
            return {"y": got[0], "h": got[1]} if c["residual"] else {"y": got}
        if c["residual"]:
            y, h = fused_rms_norm(s["x"], s["w"], residual=s["r"], eps=EPS)
            dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["r"], s["w"]), (s["gy"], s["gh"]))
            return {"y": y, "h": h, "dx": dx, "dr": dr, "dw": dw}
        y = fused_rms_norm(s["x"], s["w"], eps=EPS)
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["gy"])
        return {"y": y, "dx": dx, "dw": dw}
    with torch.no_grad():
        h, rstd, y = _norm_plain(s)
        dt = s["x"].dtype
        out = {"y": y.to(dt)}
        if c["residual"]:
            out["h"] = h.to(dt)
        if c["train"]:
            gy = s["gy"].float()
            gw = gy * s["w"].float()
            n = h * rstd
            dh = rstd * (gw - n * (gw * n).mean(dim=1, keepdim=True))
            if c["residual"]:
                dh = dh + s["gh"].float()
                out["dr"] = dh.to(dt)
            out["dx"], out["dw"] = dh.to(dt), (gy * n).sum(dim=0).to(dt)
        return out


def _groups(y, group):
    """y's rows cut into groups of columns, the last filled up with zeros."""
    rows, width = y.shape
    g = group or width
    n = -(-width // g)
    return torch.nn.functional.pad(y, (0, n * g - width)).view(rows, n, g)


def _run_fp8(s):
    c = s["case"]
    if own:
        from mlp_megakernel_b200 import fused_rms_norm_fp8

        got = fused_rms_norm_fp8(s["x"], s["w"], residual=s["r"], eps=EPS, group=c["group"])
        return dict(zip(("q", "scale", "h"), got))
    h, rstd, y = _norm_plain(s)
    b = _groups(y, c["group"])
    scale = b.abs().amax(dim=2) * (1 / E4M3_MAX)
    q = b * torch.where(scale > 0, 1 / scale, 0.0)[:, :, None]
    q = q.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(c["rows"], -1)[:, :c["width"]].contiguous()
    return {"q": q, "scale": scale, "h": h.to(s["x"].dtype)} if c["residual"] else {"q": q, "scale": scale}


def _sorted_rows(ids, experts):
    """(row of each slot, first row of each expert): stable, the slots of no expert last."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.argsort(key, stable=True)
    row = torch.empty_like(order)
    row[order] = torch.arange(order.numel(), device=ids.device)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, key, torch.ones_like(key))
    first = torch.cumsum(counts, 0) - counts
    return row.view(ids.shape), first


def _run_experts(s):
    c = s["case"]
    if own:
        from mlp_megakernel_b200 import expert_combine, expert_dispatch, expert_sort

        plan = expert_sort(s["ids"], c["experts"])
        xs = expert_dispatch(s["x"], plan)
        out = expert_combine(s["y"], s["w"], plan)
        got = {"row_of": plan.row_of, "offsets": plan.offsets, "xs": xs, "out": out}
        if c["train"]:
            got["dx"], got["dy"], got["dw"] = torch.autograd.grad((xs, out), (s["x"], s["y"], s["w"]), (s["gxs"], s["gout"]))
        return got
    with torch.no_grad():
        T, K, D = c["tokens"], c["top"], c["width"]
        dt = s["x"].dtype
        row, first = _sorted_rows(s["ids"], c["experts"])
        kept = (row < first[-1])[:, :, None]
        at = row.view(-1)
        x, w = s["x"], s["w"].float()
        xs = torch.empty_like(s["y"])
        xs[at] = torch.where(kept, x[:, None, :], 0).view(T * K, D)
        y = torch.where(kept, s["y"][at].view(T, K, D), 0).float()
        got = {"row_of": row.int(), "offsets": first.int(), "xs": xs, "out": (w[:, :, None] * y).sum(dim=1).to(dt)}
        if c["train"]:
            gout = s["gout"].float()[:, None, :]
            got["dx"] = torch.where(kept, s["gxs"][at].view(T, K, D), 0).float().sum(dim=1).to(dt)
            dy = torch.empty_like(s["y"])
            dy[at] = torch.where(kept, w[:, :, None] * gout, 0).to(dt).view(T * K, D)
            got["dy"], got["dw"] = dy, (y * gout).sum(dim=2)
        return got


def _run_adamw(s):
    c = s["case"]
    if own:
        s["opt"].step()
        return {"p": s["p"], **s["opt"].flat_state()[0]}
    s["t"] += 1
    g = s["g"].float()
    if c["bits"] == 8:
        m = (s["m"].float().view(-1, BLOCK) * s["ms"][:, None]).view(-1)
        v = (s["r"].float().view(-1, BLOCK) * s["rs"][:, None]).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    r = v.sqrt()
    step = LR / (1 - BETA1 ** s["t"]) * (m / (r / (1 - BETA2 ** s["t"]) ** 0.5 + ADAM_EPS))
    p = (s["master"] if c["master"] else s["p"].float()) * (1 - LR * DECAY) - step
    got = {"p": s["p"].copy_(p)}
    if c["master"]:
        got["master_param"] = s["master"] = p
    if c["bits"] == 8:
        (s["m"], s["ms"]), (s["r"], s["rs"]) = _quantize(m, 0.0), _quantize(r, E4M3_TINY)
        return {**got, "exp_avg": s["m"], "exp_avg_scale": s["ms"], "exp_avg_rms": s["r"], "exp_avg_rms_scale": s["rs"]}
    s["m"], s["v"] = m, v
    return {**got, "exp_avg": m, "exp_avg_sq": v}


RUN = {"norm": _run_norm, "fp8": _run_fp8, "experts": _run_experts, "adamw": _run_adamw}


def run(state):
    return RUN[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    z = SIZE[case["dtype"]]
    if case["op"] in ("norm", "fp8"):
        n, width, res = case["rows"] * case["width"], case["width"], case["residual"]
        if case["op"] == "fp8":
            g = case["group"] or width
            return {"bytes": n * (z * (3 if res else 1) + 1) + width * z + 4 * case["rows"] * -(-width // g), "flops": 7 * n}
        if not case["train"]:
            return {"bytes": n * z * (4 if res else 2) + width * z, "flops": 5 * n}
        # forward: x, (r) in, y, (h) out; backward: h, gy, (gh) in, one gradient of x and of r out
        return {"bytes": n * z * (8 if res else 5) + 3 * width * z, "flops": 16 * n}
    if case["op"] == "experts":
        T, slots, D = case["tokens"], case["tokens"] * case["top"], case["width"]
        slot = (8 if case["ids"] == "i64" else 4) + 4 + 4  # id, row, weight
        if not case["train"]:
            return {"bytes": (2 * T + 2 * slots) * D * z + slots * slot, "flops": 2 * slots * D}
        return {"bytes": (4 * T + 5 * slots) * D * z + slots * (slot + 4), "flops": 6 * slots * D}
    n = sum(_numels(case["shapes"]))
    each = (2 * z + 8 if case["master"] else 3 * z) + (4 if case["bits"] == 8 else 16)
    return {"bytes": n * each + (16 * -(-n // BLOCK) if case["bits"] == 8 else 0), "flops": 14 * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def _e4m3(v):
    """v rounded to the nearest value of the 8-bit type (4 exponent bits, 3 of mantissa, ties to even), in 64 bits."""
    _, e = torch.frexp(v)
    unit = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return (torch.round(v / unit) * unit).clamp(-E4M3_MAX, E4M3_MAX)


def _blocks64(v, width, least):
    """(8-bit values, scales) of v's rows in groups of `width`."""
    scale = v.abs().amax(dim=-1) / E4M3_MAX
    q = torch.where(scale[..., None] > 0, v / scale[..., None].clamp(min=1e-300), 0.0)
    if least:
        q = torch.where(v > 0, q.clamp(min=least), q)
    return _e4m3(q), scale


def _exact_norm(c, s):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    h = x + s["r"].detach().double() if c["residual"] else x
    rstd = (h.pow(2).sum(dim=1, keepdim=True) / c["width"] + EPS).pow(-0.5)
    y = h * rstd * w
    if c["op"] == "fp8":
        q, scale = _blocks64(_groups(y, c["group"]), None, 0.0)
        got = {"q": q.view(c["rows"], -1)[:, :c["width"]], "scale": scale}
        return {**got, "h": h} if c["residual"] else got
    got = {"y": y}
    if c["residual"]:
        got["h"] = h
    if c["train"]:
        gy = s["gy"].double()
        dh = rstd * gy * w - h * rstd.pow(3) * ((gy * w * h).sum(dim=1, keepdim=True) / c["width"])
        if c["residual"]:
            dh = dh + s["gh"].double()
            got["dr"] = dh
        got["dx"], got["dw"] = dh, (gy * h * rstd).sum(dim=0)
    return got


def _exact_experts(c, s):
    T, K, E, D = c["tokens"], c["top"], c["experts"], c["width"]
    ids = s["ids"].reshape(-1).long().cpu()
    ids = torch.where((ids < 0) | (ids >= E), E, ids)
    slots = torch.cat([torch.nonzero(ids == e)[:, 0] for e in range(E + 1)]).cuda()  # the slot of each row
    kept = int((ids < E).sum())
    slots = slots[:kept]
    token = slots // K
    x, y, w = s["x"].detach().double(), s["y"].detach().double(), s["w"].detach().double().reshape(-1)
    xs = torch.zeros(T * K, D, dtype=torch.float64, device="cuda")
    xs[:kept] = x[token]
    got = {"row_of": None, "offsets": None, "xs": xs,
           "out": torch.zeros_like(x).index_add_(0, token, y[:kept] * w[slots, None])}
    if c["train"]:
        gout = s["gout"].double()[token]
        got["dx"] = torch.zeros_like(x).index_add_(0, token, s["gxs"].double()[:kept])
        got["dy"], got["dw"] = torch.zeros_like(xs), torch.zeros_like(w)
        got["dy"][:kept] = gout * w[slots, None]
        got["dw"][slots] = (gout * y[:kept]).sum(dim=1)
        got["dw"] = got["dw"].view(T, K)
    return got


def _exact_adamw(c, s):
    g, p, t = s["g"].double(), s["master" if c["master"] else "p"].double(), STEP + 1
    if c["bits"] == 8:
        m = (s["m"].double().view(-1, BLOCK) * s["ms"].double()[:, None]).view(-1)
        v = (s["r"].double().view(-1, BLOCK) * s["rs"].double()[:, None]).view(-1).pow(2)
    else:
        m, v = s["m"].double(), s["v"].double()
    m, v = BETA1 * m + (1 - BETA1) * g, BETA2 * v + (1 - BETA2) * g.pow(2)
    mean, square = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = p - LR * DECAY * p - LR * mean / (square.sqrt() + ADAM_EPS)
    got = {"p": p, "master_param": p} if c["master"] else {"p": p}
    if c["bits"] == 32:
        return {**got, "exp_avg": m, "exp_avg_sq": v}
    (mq, ms), (rq, rs) = _blocks64(m.view(-1, BLOCK), BLOCK, 0.0), _blocks64(v.sqrt().view(-1, BLOCK), BLOCK, E4M3_TINY)
    return {**got, "exp_avg": mq.view(-1), "exp_avg_scale": ms, "exp_avg_rms": rq.view(-1), "exp_avg_rms_scale": rs}


def exact(case, seed):
    global own
    was, own = own, False  # the inputs alone
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"norm": _exact_norm, "fp8": _exact_norm, "experts": _exact_experts, "adamw": _exact_adamw}[case["op"]](case, s)
