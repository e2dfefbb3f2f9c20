"""What is measured of the feed-forward operators: the matrix product with bias, activation and residual, the gated
feed-forward block, and activation checkpoints in 8 bits with their use in both backward passes.

Each operator has a plain form in elementary torch operations (fp32 throughout, one rounding at the end) next to the
call of the framework's own kernels, and a statement of its definition in 64 bits (``exact``).
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
E4M3_MAX = 448.0
GROUP = 128  # columns that share a scale of a checkpoint
TINY = 2.0 ** -126  # the smallest scale
GELU_A, GELU_B = math.sqrt(2 / math.pi), 0.044715


def listed():
    return [
        # an output projection at a decoding step: latency and the weights' bytes
        dict(name="linear_one_row", op="linear", rows=1, d_in=4096, d_out=4096, dtype="bf16", act=None, bias=True, residual=True, train=False, bits=16),
        # a decoding batch through a wide layer
        dict(name="linear_batch", op="linear", rows=48, d_in=4096, d_out=14336, dtype="bf16", act="gelu_tanh", bias=True, residual=False, train=False, bits=16),
        # an output projection over a long prompt
        dict(name="linear_prompt", op="linear", rows=8192, d_in=4096, d_out=4096, dtype="bf16", act=None, bias=False, residual=True, train=False, bits=16),
        # training rows and widths that no tile divides
        dict(name="linear_train_odd", op="linear", rows=5003, d_in=1000, d_out=2056, dtype="f16", act="gelu_tanh", bias=True, residual=True, train=True, bits=16),
        # a wide layer's training batch, its saved activations in 8 bits
        dict(name="linear_train_8bit", op="linear", rows=16384, d_in=2048, d_out=8192, dtype="bf16", act="silu", bias=True, residual=False, train=True, bits=8),
        # one token's feed-forward block at a decoding step
        dict(name="gated_one_row", op="gated", rows=1, d_in=4096, hidden=14336, dtype="bf16", act="silu", residual=True, train=False, bits=16),
        # the fused MLP's widest network, gated, on a small batch: latency
        dict(name="gated_small", op="gated", rows=64, d_in=256, hidden=256, dtype="f16", act="softplus", residual=False, train=False, bits=16),
        # a prompt of a length that no tile divides
        dict(name="gated_prompt", op="gated", rows=3001, d_in=4096, hidden=11008, dtype="bf16", act="silu", residual=True, train=False, bits=16),
        # a training batch's feed-forward block
        dict(name="gated_train", op="gated", rows=16384, d_in=4096, hidden=11008, dtype="bf16", act="silu", residual=True, train=True, bits=16),
        # a narrower one with an odd number of rows, its saved activations in 8 bits
        dict(name="gated_train_8bit", op="gated", rows=20011, d_in=1024, hidden=2816, dtype="f16", act="gelu_tanh", residual=True, train=True, bits=8),
        # a training batch's activations kept in 8 bits for a backward pass of the user's own
        dict(name="checkpoint", op="checkpoint", rows=16384, width=8192, dtype="bf16"),
        # rows that no vector load divides
        dict(name="checkpoint_odd", op="checkpoint", rows=5003, width=1999, dtype="f16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def _width(rng, low, high):
    """A multiple of 8; of 64 half of the time."""
    unit = rng.choice([8, 64])
    return max(unit, _log(rng, low, high) // unit * unit)


def draw(rng):
    op = rng.choice(["linear", "linear", "gated", "gated", "checkpoint"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "checkpoint":
        width = _log(rng, 8, 16384)
        return dict(op=op, rows=_log(rng, 1, min(131072, (1 << 27) // width)), width=width, dtype=rng.choice(["f16", "bf16", "f32"]))
    train = rng.random() < 0.6
    case = dict(op=op, d_in=_width(rng, 16, 8192), dtype=dtype, act=rng.choice(["relu", "silu", "gelu_tanh", "softplus", "sigmoid"]),
                residual=rng.random() < 0.5, train=train, bits=rng.choice([8, 16]) if train else 16)
    if op == "linear":
        case.update(d_out=_width(rng, 16, 14336), bias=rng.random() < 0.5)
        if rng.random() < 0.3:
            case["act"] = None
        each = case["d_in"] * case["d_out"]
    else:
        case["hidden"] = _width(rng, 16, 14336)
        each = 3 * case["d_in"] * case["hidden"]
    return {**case, "rows": _log(rng, 1, min(65536, 2 * 10 ** 12 // each))}


def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, scale, generator=g)

    return normal


def prepare(case, seed):
    normal, dt, rows = _random(seed), DTYPES[case["dtype"]], case["rows"]
    if case["op"] == "checkpoint":
        # rows of a norm's output: most values near 1, a few columns much larger
        return {"case": case, "x": normal(rows, case["width"], dtype=dt) * (1 + 20 * (normal(case["width"]).abs() > 2.5)).to(dt)}
    k = case["d_in"]
    s = {"case": case, "x": normal(rows, k, dtype=dt)}
    if case["op"] == "linear":
        n, leaves = case["d_out"], ["x", "w"]
        s["w"] = normal(k, n, dtype=dt, scale=k ** -0.5)
        s["b"] = normal(n, dtype=dt, scale=0.5) if case["bias"] else None
        leaves += ["b"] if case["bias"] else []
    else:
        n, h, leaves = k, case["hidden"], ["x", "wg", "wu", "wd"]
        s["wg"], s["wu"] = normal(k, h, dtype=dt, scale=k ** -0.5), normal(k, h, dtype=dt, scale=k ** -0.5)
        s["wd"] = normal(h, n, dtype=dt, scale=h ** -0.5)
    s["r"] = normal(rows, n, dtype=dt, scale=2.0) if case["residual"] else None
    if case["train"]:
        s["go"] = normal(rows, n, dtype=dt, scale=0.1)
        for name in leaves:
            s[name].requires_grad_(True)
    return s


# ---------------------------------------------------------------- plain forms
def _act(kind, z):
    if kind is None:
        return z
    if kind == "relu":
        return z.clamp(min=0)
    if kind == "softplus":
        return z.clamp(min=0) + torch.log1p(torch.exp(-z.abs()))
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2 * GELU_A * (z + GELU_B * z * z * z))
    s = torch.sigmoid(z)
    return s if kind == "sigmoid" else z * s


def _slope(kind, z):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu_tanh":
        s = torch.sigmoid(2 * GELU_A * (z + GELU_B * z * z * z))
        return s + z * s * (1 - s) * (2 * GELU_A * (1 + 3 * GELU_B * z * z))
    s = torch.sigmoid(z)
    return {"softplus": s, "sigmoid": s * (1 - s), "silu": s + z * s * (1 - s)}[kind]


def _in_8_bits(v):
    """(8-bit values, scales [rows, groups]) of v's rows in groups of GROUP columns: the scale is the smallest power of
    two that brings the group's largest magnitude to 448 at most."""
    rows, width = v.shape
    n = -(-width // GROUP)
    b = torch.nn.functional.pad(v, (0, n * GROUP - width)).view(rows, n, GROUP)
    most = b.abs().amax(dim=2)
    m, e = torch.frexp(most / E4M3_MAX)
    scale = torch.ldexp(torch.ones_like(most), torch.where(m > 0.5, e, e - 1))
    scale = torch.where(most > 0, scale, 0.0).clamp(min=TINY)
    return (b / scale[:, :, None]).to(torch.float8_e4m3fn), scale


def _from_8_bits(q, scale, width):
    return (q.float() * scale[:, :, None]).view(q.shape[0], -1)[:, :width]


def _kept(v, bits):
    """What the backward pass has of v."""
    return v if bits == 16 else _from_8_bits(*_in_8_bits(v), v.shape[1])


def _run_linear(s):
    c = s["case"]
    if own:
        from mlp_megakernel_b200 import fused_linear

        kept = torch.float8_e4m3fn if c["bits"] == 8 else None
        out = fused_linear(s["x"], s["w"], s["b"], activation=c["act"], residual=s["r"], activation_dtype=kept)
        if not c["train"]:
            return {"out": out}
        grads = torch.autograd.grad(out, [s["x"], s["w"]] + ([s["b"]] if c["bias"] else []), s["go"])
        return {"out": out, **dict(zip(("dx", "dw", "db"), grads))}
    with torch.no_grad():
        dt, x, w = s["x"].dtype, s["x"].float(), s["w"].float()
        z = x @ w
        if c["bias"]:
            z = z + s["b"].float()
        out = _act(c["act"], z)
        if c["residual"]:
            out = out + s["r"].float()
        got = {"out": out.to(dt)}
        if c["train"]:
            dz = s["go"].float()
            if c["act"] is not None:
                dz = dz * _slope(c["act"], _kept(z, c["bits"]))
            got["dx"], got["dw"] = (dz @ w.t()).to(dt), (_kept(x, c["bits"]).t() @ dz).to(dt)
            if c["bias"]:
                got["db"] = dz.sum(dim=0).to(dt)
        return got


def _run_gated(s):
    c = s["case"]
    if own:
        from mlp_megakernel_b200 import fused_gated_mlp

        kept = torch.float8_e4m3fn if c["bits"] == 8 else None
        out = fused_gated_mlp(s["x"], s["wg"], s["wu"], s["wd"], activation=c["act"], residual=s["r"], activation_dtype=kept)
        if not c["train"]:
            return {"out": out}
        grads = torch.autograd.grad(out, [s["x"], s["wg"], s["wu"], s["wd"]], s["go"])
        return {"out": out, **dict(zip(("dx", "dwg", "dwu", "dwd"), grads))}
    with torch.no_grad():
        dt = s["x"].dtype
        x, wg, wu, wd = (s[k].float() for k in ("x", "wg", "wu", "wd"))
        g, u = x @ wg, x @ wu
        h = _act(c["act"], g) * u
        out = h @ wd
        if c["residual"]:
            out = out + s["r"].float()
        got = {"out": out.to(dt)}
        if c["train"]:
            go = s["go"].float()
            if c["bits"] == 8:
                x, g, u = _kept(x, 8), _kept(g, 8), _kept(u, 8)
                h = _act(c["act"], g) * u
            dh = go @ wd.t()
            du, dg = dh * _act(c["act"], g), dh * u * _slope(c["act"], g)
            got["dx"] = (dg @ wg.t() + du @ wu.t()).to(dt)
            got["dwg"], got["dwu"], got["dwd"] = (x.t() @ dg).to(dt), (x.t() @ du).to(dt), (h.t() @ go).to(dt)
        return got


def _run_checkpoint(s):
    x = s["x"]
    if own:
        from mlp_megakernel_b200 import fp8_checkpoint, fp8_restore

        q, scale = fp8_checkpoint(x)
        return {"scale": scale, "back": fp8_restore(q, scale, x.dtype)}
    q, scale = _in_8_bits(x.float())
    return {"scale": scale, "back": _from_8_bits(q, scale, x.shape[1]).to(x.dtype)}


RUN = {"linear": _run_linear, "gated": _run_gated, "checkpoint": _run_checkpoint}


def run(state):
    return RUN[state["case"]["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without
def _checkpoint_bytes(rows, width):
    return rows * (width + 4 * -(-width // GROUP))


def work(case):
    z, rows = SIZE[case["dtype"]], case["rows"]
    if case["op"] == "checkpoint":
        n = rows * case["width"]
        return {"bytes": 2 * (n * z + _checkpoint_bytes(rows, case["width"])), "flops": 3 * n}
    k = case["d_in"]
    saved = (lambda width: _checkpoint_bytes(rows, width)) if case["bits"] == 8 else (lambda width: rows * width * z)
    if case["op"] == "linear":
        n = case["d_out"]
        weights, kept, flops = k * n + (n if case["bias"] else 0), saved(n) if case["act"] else 0, 2 * rows * k * n
    else:
        n, h = k, case["hidden"]
        weights, kept, flops = 2 * k * h + h * n, 2 * saved(h), 2 * rows * h * (2 * k + n)
    rows_in_and_out = rows * (k + n * (2 if case["residual"] else 1))
    if not case["train"]:
        return {"bytes": z * (rows_in_and_out + weights), "flops": flops}
    if case["bits"] == 8:
        kept += saved(k)  # the input's checkpoint
    return {"bytes": z * (rows_in_and_out + rows * (n + k) + 2 * weights) + 2 * kept, "flops": 3 * flops}


# ---------------------------------------------------------------- the definitions in 64 bits
def _act64(kind, z):
    """(the activation, its derivative), written with the hyperbolic tangent and the exponential's own forms."""
    one = torch.ones_like(z)
    if kind is None:
        return z, one
    if kind == "relu":
        return torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).to(z.dtype)
    if kind == "gelu_tanh":
        t = torch.tanh(GELU_A * (z + GELU_B * z.pow(3)))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * GELU_A * (1 + 3 * GELU_B * z.pow(2))
    s = 0.5 * (1 + torch.tanh(0.5 * z))
    s = torch.where(z < -20, torch.exp(z.clamp(max=0)), s)  # 1 + tanh loses what is left there; off by exp(-20) at most
    if kind == "sigmoid":
        return s, s * (one - s)
    if kind == "silu":
        return z * s, s * (one + z * (one - s))
    return torch.where(z > 0, z + torch.log1p(torch.exp(-z.clamp(min=0))), torch.log1p(torch.exp(z.clamp(max=0)))), s


def _checkpoint64(v):
    """(values that the 8-bit numbers stand for, scales), each group cut out by itself."""
    parts, scales = [], []
    for part in v.split(GROUP, dim=1):
        most = part.abs().amax(dim=1, keepdim=True)
        power = torch.ceil(torch.log2(torch.where(most > 0, most, 1.0) / E4M3_MAX))
        # log2 may be off at a border
        power = power + (most > E4M3_MAX * torch.exp2(power)).double() - (most <= E4M3_MAX * torch.exp2(power - 1)).double()
        scale = torch.where(most > 0, torch.exp2(power), TINY).clamp(min=TINY)
        y = part / scale
        _, e = torch.frexp(y)
        unit = torch.ldexp(torch.ones_like(y), (e - 4).clamp(min=-9))  # 4 binary digits, 2^-9 at least
        parts.append(torch.round(y / unit) * unit * scale)
        scales.append(scale)
    return torch.cat(parts, dim=1), torch.cat(scales, dim=1)


def _exact_linear(c, s):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    z = torch.mm(x, w)
    if c["bias"]:
        z += s["b"].detach().double()
    out = _act64(c["act"], z)[0]
    got = {"out": out + s["r"].double() if c["residual"] else out}
    if c["train"]:
        dz = s["go"].double()
        if c["bits"] == 8:
            x, z = _checkpoint64(x)[0], _checkpoint64(z)[0]
        dz = dz * _act64(c["act"], z)[1]
        got["dx"], got["dw"] = torch.mm(dz, w.t()), torch.mm(x.t(), dz)
        if c["bias"]:
            got["db"] = torch.mm(torch.ones(1, c["rows"], device=x.device, dtype=x.dtype), dz)[0]
    return got


def _exact_gated(c, s):
    x, wg, wu, wd = (s[k].detach().double() for k in ("x", "wg", "wu", "wd"))
    both = torch.mm(x, torch.cat([wg, wu], dim=1))
    g, u = both[:, :c["hidden"]], both[:, c["hidden"]:]
    out = torch.mm(_act64(c["act"], g)[0] * u, wd)
    got = {"out": out + s["r"].double() if c["residual"] else out}
    if c["train"]:
        go = s["go"].double()
        if c["bits"] == 8:
            x, g, u = _checkpoint64(x)[0], _checkpoint64(g)[0], _checkpoint64(u)[0]
        a, slope = _act64(c["act"], g)
        dh = torch.mm(go, wd.t())
        both = torch.cat([dh * u * slope, dh * a], dim=1)
        got["dx"] = torch.mm(both, torch.cat([wg, wu], dim=1).t())
        dw = torch.mm(x.t(), both)
        got["dwg"], got["dwu"] = dw[:, :c["hidden"]], dw[:, c["hidden"]:]
        got["dwd"] = torch.mm((a * u).t(), go)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "checkpoint":
        back, scale = _checkpoint64(s["x"].double())
        return {"scale": scale, "back": back}
    return (_exact_linear if case["op"] == "linear" else _exact_gated)(case, s)
