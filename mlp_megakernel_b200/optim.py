"""AdamW over many tensors in one launch, with the state in 32 bits or in 8
(no counterpart in the reference, which leaves the step to its caller).

``FusedAdamW`` is a ``torch.optim.Optimizer``: learning-rate schedulers,
parameter groups, ``state_dict``, its hooks and GradScaler work as with torch's
AdamW.  (What differs: ``state[p]`` holds parts of flat buffers, to be read and
written in place, and has no ``step``, which is in ``state_dict`` alone.)
All tensors of a parameter group that share their types are stepped by one
kernel launch on the current CUDA stream (768 tensors at most each); there is
no CPU path.
"""
from __future__ import annotations

import bisect

import torch
from torch import Tensor

from . import _lib
from ._native import native
from .norm import DTYPES

BLOCK = _lib.ADAMW_BLOCK


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def _dense(t: Tensor) -> bool:
    """Whether the elements fill one stretch of memory, in any order of the
    dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for size, stride in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n != 1), key=lambda d: d[1]):
        if stride != want:
            return False
        want *= size
    return True


class _Bucket:
    """The flat state of some tensors that got it together: each begins at a
    multiple of BLOCK elements, and what pads it is zero.  `group` is the place of
    the parameter group that they were in."""

    def __init__(self, params, group: int, bits: int, master: bool):
        self.params, self.group, self.bits = list(params), group, bits
        self.numel = [p.numel() for p in self.params]
        self.off, total = [], 0
        for n in self.numel:
            self.off.append(total)
            total += _blocks(n) * BLOCK
        dev = self.params[0].device
        total = max(total, BLOCK)  # tensors of no elements have a state too

        def zeros(n, dtype):
            return torch.zeros(n, device=dev, dtype=dtype)

        if bits == 8:
            self.flat = {"exp_avg": zeros(total, torch.float8_e4m3fn), "exp_avg_scale": zeros(total // BLOCK, torch.float32),
                         "exp_avg_rms": zeros(total, torch.float8_e4m3fn),
                         "exp_avg_rms_scale": zeros(total // BLOCK, torch.float32)}
        else:
            self.flat = {"exp_avg": zeros(total, torch.float32), "exp_avg_sq": zeros(total, torch.float32)}
        if master:
            self.flat["master_param"] = zeros(total, torch.float32)
        self.ticks = torch.zeros(len(self.params), device=dev, dtype=torch.int64)
        self.chunks = [max(1, -(-n // _lib.ADAMW_CHUNK)) for n in self.numel]
        if master:
            for i, p in enumerate(self.params):
                self.view(i, "master_param").copy_(p.detach())

    def launch(self, members):
        """What steps the members (their places in this bucket) in one go."""
        sq = self.flat["exp_avg_rms" if self.bits == 8 else "exp_avg_sq"]
        return native().AdamwBucket(
            [self.params[i] for i in members], [self.off[i] for i in members], list(members), self.bits,
            self.flat["exp_avg"], sq, self.flat.get("exp_avg_scale"), self.flat.get("exp_avg_rms_scale"),
            self.flat.get("master_param"), self.ticks)

    def view(self, i: int, name: str) -> Tensor:
        """Tensor i's part of a flat buffer: of its own shape and strides, or
        [blocks] for a scale."""
        flat = self.flat[name]
        if name.endswith("_scale"):
            return flat[self.off[i] // BLOCK:self.off[i] // BLOCK + _blocks(self.numel[i])]
        p = self.params[i]
        return flat[self.off[i]:self.off[i] + self.numel[i]].as_strided(p.shape, p.stride(),
                                                                         flat.storage_offset() + self.off[i])

    def steps(self) -> list:
        return [int(t) // c for t, c in zip(self.ticks.tolist(), self.chunks)]


class _Plan:
    """What a step of one parameter group does, as long as the group holds the same
    parameters: the launches, and the parameters that have no state yet."""

    def __init__(self, group, params, launches, waiting):
        self.group, self.params, self.launches, self.waiting = group, params, launches, waiting


class FusedAdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) for CUDA parameters in fp32, fp16 or bf16.

    ``state_bits=32`` keeps m and v in fp32.  ``state_bits=8`` keeps m and sqrt(v)
    as e4m3 in blocks of 256 elements with an fp32 scale each: 2.03 bytes an
    element instead of 8.  (Blocks are of a tensor's elements in memory order.  A
    gradient that is not finite makes its whole block's state NaN: use GradScaler
    or clip.)  ``master_weights=True`` keeps an fp32 copy of each 16-bit
    parameter, made when its state is, which is stepped and rounded into the
    parameter (what else is written into the parameter later is lost); without it
    a 16-bit parameter is stepped in fp32 and rounded to itself, as in torch.  ``lr`` is a number or a CUDA tensor of one element.

    A step is over what the parameter groups hold then: a parameter that moves to
    another group keeps its state, one taken out is left as it is, and one whose
    entry of ``state`` is deleted begins anew.  A parameter whose ``grad`` is None is
    left as it is.  Gradients are in the parameter's dtype or fp32.  The step count
    is on the device, so ``step()`` can be captured in a CUDA graph after one
    ordinary step, and a step that GradScaler's ``found_inf`` skips does not count.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *,
                 state_bits: int = 32, master_weights: bool = False, maximize: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, maximize=maximize)
        self._state_bits, self._master = state_bits, master_weights
        self._buckets: list = []  # in the order of their groups
        self._place: dict = {}    # parameter: (bucket, its place there, its dict in self.state)
        self._plans: dict = {}    # id of a parameter group: _Plan
        self._known = 0           # entries of self.state when it was looked through
        self._step_supports_amp_scaling = True
        super().__init__(params, defaults)

    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_group(group) -> None:
        lr, (b1, b2) = group["lr"], group["betas"]
        if isinstance(lr, Tensor):
            if lr.numel() != 1 or lr.dtype != torch.float32 or not lr.is_cuda:
                raise ValueError("a tensor lr must be one float32 value on the GPU")
        elif not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be at least 0 and below 1, got {(b1, b2)}")
        if not group["eps"] >= 0.0 or not group["weight_decay"] >= 0.0:
            raise ValueError("eps and weight_decay must not be negative")
        FusedAdamW._check_once(group["params"])
        FusedAdamW._check_params(group["params"])

    @staticmethod
    def _check_once(params) -> None:
        if len({id(p) for p in params}) != len(params):  # its steps would be one launch's, over the same values
            raise ValueError("a parameter group holds a parameter twice")

    @staticmethod
    def _check_params(params) -> None:
        for p in params:
            if not p.is_cuda:
                raise RuntimeError("FusedAdamW runs on CUDA (sm_100) only; got a CPU parameter")
            if p.dtype not in DTYPES:
                raise TypeError(f"FusedAdamW takes fp16, bf16 or fp32 parameters; got {p.dtype}")
            if not _dense(p):
                raise ValueError(f"a parameter of shape {tuple(p.shape)} and strides {p.stride()} does not fill its memory")

    def _add_state(self, g: int, params) -> None:
        """State for parameters of group g that have none, a bucket for each type
        and device."""
        kinds: dict = {}
        for p in params:
            kinds.setdefault((p.dtype, p.device), []).append(p)
        for (dtype, dev), ps in kinds.items():
            with torch.cuda.device(dev):
                b = _Bucket(ps, g, self._state_bits, self._master and dtype != torch.float32)
            bisect.insort(self._buckets, b, key=lambda b: b.group)
            for i, p in enumerate(ps):
                self.state[p] = {name: b.view(i, name) for name in b.flat}
                self._place[p] = (b, i, self.state[p])
        self._known = len(self.state)

    def _look_through_state(self) -> None:
        """Parameters whose state was taken out of self.state have none."""
        self._place = {p: place for p, place in self._place.items() if self.state.get(p) is place[2]}
        left = {id(b) for b, *_ in self._place.values()}
        self._buckets = [b for b in self._buckets if id(b) in left]
        self._plans.clear()
        self._known = len(self.state)

    def _plan(self, g: int, group) -> _Plan:
        """The plan of group g: made anew when its list of parameters has changed, or
        when one without state has got its first gradient."""
        plan, params = self._plans.get(id(group)), group["params"]
        if plan is not None and native().same_items(plan.params, params) and \
                not (plan.waiting and any(p.grad is not None for p in plan.waiting)):
            return plan
        self._check_once(params)
        new = [p for p in params if p not in self._place and p.grad is not None]
        self._check_params(new)
        self._add_state(g, new)
        return self._make_plan(group)

    def _make_plan(self, group) -> _Plan:
        params = group["params"]
        members: dict = {}  # of each bucket
        for p in params:
            if p in self._place:
                b, i, _ = self._place[p]
                members.setdefault(id(b), (b, []))[1].append(i)
        plan = _Plan(group, list(params), [b.launch(m) for b, m in members.values()],
                     [p for p in params if p not in self._place])
        groups = {id(other) for other in self.param_groups}
        self._plans = {k: v for k, v in self._plans.items() if k in groups}
        self._plans[id(group)] = plan
        return plan

    def step(self, closure=None, *, grad_scale=None, found_inf=None):
        """One step.  ``grad_scale`` and ``found_inf`` (fp32 values on the GPU, as
        GradScaler passes them): the gradients are divided by the one; a
        ``found_inf`` that is not 0 leaves parameters, state and step count as
        they were."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        grad_scale = getattr(self, "grad_scale", None) if grad_scale is None else grad_scale
        found_inf = getattr(self, "found_inf", None) if found_inf is None else found_inf
        if len(self.state) != self._known:
            self._look_through_state()
        for g, group in enumerate(self.param_groups):
            launches = self._plan(g, group).launches
            lr, (b1, b2) = group["lr"], group["betas"]
            lr, lr_tensor = (0.0, lr) if isinstance(lr, Tensor) else (lr, None)
            for launch in launches:
                launch.step(lr, lr_tensor, b1, b2, group["eps"], group["weight_decay"], group["maximize"], grad_scale,
                            found_inf)
        return loss

    def __reduce__(self):
        raise TypeError("FusedAdamW is saved and copied by its state_dict()")

    # ------------------------------------------------------------ state
    def flat_state(self) -> list:
        """The state's own buffers, a dict for each group and type of tensors in
        the order they got their state (each in the group that it had then): ``exp_avg`` and ``exp_avg_sq`` (32 bits), or
        ``exp_avg``, ``exp_avg_scale``, ``exp_avg_rms`` and ``exp_avg_rms_scale``
        (8 bits), and ``master_param``.  A tensor's part begins at a multiple of
        256 elements; what pads it is zero."""
        return [b.flat for b in self._buckets]

    def state_dict(self) -> dict:
        """As torch's, hooks included: ``state[i]`` has ``step`` (a number; the host
        waits for the GPU) and the tensors of parameter i, ``param_groups`` the rest."""
        for hook in list(self._optimizer_state_dict_pre_hooks.values()):
            hook(self)
        if len(self.state) != self._known:
            self._look_through_state()
        number, groups = {}, []
        for group in self.param_groups:
            packed = {k: v for k, v in group.items() if k != "params"}
            packed["params"] = [number.setdefault(p, len(number)) for p in group["params"]]
            groups.append(packed)
        steps = {id(b): b.steps() for b in self._buckets}
        state = {}
        for p, n in number.items():
            if p in self._place:
                b, i, _ = self._place[p]
                state[n] = {"step": steps[id(b)][i], **{name: b.view(i, name) for name in b.flat}}
        found = {"state": state, "param_groups": groups}
        for hook in list(self._optimizer_state_dict_post_hooks.values()):
            got = hook(self, found)
            found = found if got is None else got
        return found

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """Takes what ``state_dict`` gave, of the same ``state_bits`` and
        ``master_weights``; the values are copied, from any device.  A load that is
        refused changes nothing.  Hooks are called as torch's optimizers call them."""
        state_dict = state_dict.copy()
        for hook in list(self._optimizer_load_state_dict_pre_hooks.values()):
            got = hook(self, state_dict)
            state_dict = state_dict if got is None else got
        groups, state = state_dict["param_groups"], state_dict["state"]
        if len(groups) != len(self.param_groups) or \
                any(len(a["params"]) != len(b["params"]) for a, b in zip(groups, self.param_groups)):
            raise ValueError("the state is of other parameter groups")
        loads = []
        for g, (saved, group) in enumerate(zip(groups, self.param_groups)):
            found = [(p, state[i]) for i, p in zip(saved["params"], group["params"]) if i in state]
            for p, s in found:
                names = {"exp_avg", "exp_avg_scale", "exp_avg_rms", "exp_avg_rms_scale"} if self._state_bits == 8 else \
                    {"exp_avg", "exp_avg_sq"}
                names |= {"master_param"} if self._master and p.dtype != torch.float32 else set()
                if set(s) != names | {"step"}:
                    raise ValueError(f"the state of a parameter holds {sorted(s)}, expected {sorted(names | {'step'})}")
                if int(s["step"]) < 0:
                    raise ValueError(f"a step count must not be negative, got {s['step']}")
                for name in names:
                    n = _blocks(p.numel()) if name.endswith("_scale") else p.numel()
                    kind = torch.float8_e4m3fn if self._state_bits == 8 and name in ("exp_avg", "exp_avg_rms") else \
                        torch.float32
                    if s[name].numel() != n or s[name].dtype != kind:
                        raise ValueError(f"{name} must hold {n} values of {kind}")
            options = {k: v.clone() if isinstance(v, Tensor) else v for k, v in saved.items() if k != "params"}
            if isinstance(options.get("lr"), Tensor) and group["params"]:  # a checkpoint read to the host
                options["lr"] = options["lr"].to(group["params"][0].device)
            self._check_group({**group, **options})
            loads.append((found, options))
        # Nothing has changed so far, and nothing is refused from here on.
        self.state.clear()
        self._buckets, self._place, self._plans = [], {}, {}
        for g, (found, options) in enumerate(loads):
            self.param_groups[g].update(options)
            self._add_state(g, [p for p, _ in found])
        saved = dict(pair for found, _ in loads for pair in found)
        for b in self._buckets:
            for i, p in enumerate(b.params):
                for name in b.flat:
                    v = b.view(i, name)
                    v.copy_(saved[p][name].reshape(v.shape))
            b.ticks.copy_(torch.tensor([int(saved[p]["step"]) * c for p, c in zip(b.params, b.chunks)]))
        for group in self.param_groups:  # here and not in the first step
            self._make_plan(group)
        for hook in list(self._optimizer_load_state_dict_post_hooks.values()):
            hook(self)
