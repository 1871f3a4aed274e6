"""AdamW over everything a network learns, in one launch, with moments in 32 bits or in 8.

The reference's trainer (``snn_runners/trainer.py:358-384``) clips the gradients and steps
a torch optimiser. What it steps here reaches from a 41 x 40 table of type-pair scales to a
weight per synapse (hundreds of millions), where the optimiser's two moments weigh more than
the weights: ``AdamW(..., state_bits=8)`` holds them in a byte each (e4m3 codes, a float
scale per 256 elements, rounded stochastically from a seed), ``state_bits=32`` in a float
each. ``max_norm`` clips the global norm on the device, without a host read, and leaves out
a step whose norm is not finite (its squares are float32's: a gradient above 1.8e19 makes it so).
"""

from __future__ import annotations

from array import array
from itertools import chain, repeat
from operator import attrgetter, is_, is_not

import torch

from wiretorch_b200 import _lib

BLOCK = 256  # WT_ADAMW_BLOCK: elements that share a scale of the 8-bit moments
SKIPPED = 16  # offsetof(WtStepControl, skipped)
_C = _lib.C
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # WT_F32, WT_BF16, WT_F16


class _GradNorm(_C.Structure):
    _fields_ = [
        ("n", _C.c_int32), ("g", _lib.P), ("numel", _lib.P), ("type", _lib.P), ("max_norm", _C.c_float),
        ("partial", _lib.P), ("control", _lib.P),
    ]  # fmt: skip


class _AdamW(_C.Structure):
    _fields_ = [
        ("n", _C.c_int32), ("type", _C.c_int32), ("state_bits", _C.c_int32),
        ("p", _lib.P), ("g", _lib.P), ("m", _lib.P), ("v", _lib.P),
        ("m_scale", _lib.P), ("v_scale", _lib.P), ("master", _lib.P),
        ("numel", _lib.P), ("first", _lib.P), ("lr", _lib.P), ("weight_decay", _lib.P),
        ("beta1", _C.c_double), ("beta2", _C.c_double), ("eps", _C.c_double),
        ("step", _C.c_int64), ("count", _C.c_int64), ("seed", _C.c_uint64), ("control", _lib.P),
        ("skipped", _lib.P), ("before", _lib.P),
    ]  # fmt: skip


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one stretch of memory, in some order of the dimensions."""
    if t.is_contiguous():
        return True
    expected = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s != 1), key=lambda d: d[1]):
        if stride != expected:
            return False
        expected *= size
    return True


# Accessors to map over many tensors: a step looks at each of them, at some 60 ns a look.
_data_ptr, _numel, _get_device = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device
_is_contiguous, _dtype = torch.Tensor.is_contiguous, torch.Tensor.dtype.__get__
_grad = attrgetter("grad")


def _addresses(tensors):
    return array("Q", map(_data_ptr, tensors))


def _at(values):
    """The address of an array's values."""
    return values.buffer_info()[0]


def _same(a, b):
    """Whether two lists hold the same objects."""
    return len(a) == len(b) and all(map(is_, a, b))


class _Batch:
    """The tensors that one call steps, those of one type, betas and eps, with the objects that
    were checked when it was made; their addresses are read anew in every step."""

    def __init__(self, dtype, betas, eps):
        self.dtype, self.betas, self.eps = dtype, betas, eps
        self.params, self.held, self.groups, self.first, self.numel = [], [], [], [], []
        self.strided = False  # a tensor in another order than its dimensions'

    def add(self, p, held, group, first):
        self.params.append(p)
        self.held.append(held)
        self.groups.append(group)
        self.first.append(first)
        self.numel.append(p.numel())
        self.strided |= not p.is_contiguous()

    def close(self, names):
        self.state = {name: [h[name] for h in self.held] for name in names}
        self.before = [h.get("before") for h in self.held] if any("before" in h for h in self.held) else None
        self.types = array("i", [TYPES[self.dtype]]) * len(self.params)
        self.counts, self.firsts = array("q", self.numel), array("q", self.first)
        self.index = self.params[0].get_device()

    def _as_planned(self, tensors):
        n = len(tensors)
        return (all(map(_is_contiguous, tensors)) and list(map(_numel, tensors)) == self.numel
                and list(map(_dtype, tensors)).count(self.dtype) == n
                and list(map(_get_device, tensors)).count(self.index) == n)  # fmt: skip

    def is_current(self):
        """Whether the tensors are of the sizes, type and device that were checked; a batch with a
        strided tensor is checked in every step."""
        return not self.strided and self._as_planned(self.params)

    def takes(self, grads):
        """Whether the gradients can be read as they are."""
        return not self.strided and self._as_planned(grads)

    def rates(self, name):
        groups = self.groups
        if groups[0] is groups[-1]:  # they come group by group
            return array("d", [groups[0][name]]) * len(groups)
        return array("d", [group[name] for group in groups])


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over float32, bfloat16 or float16 CUDA tensors.

    ``state_bits``: 32 or 8, what each moment is held in. 16-bit tensors keep a float32
    master among their state, made from the tensor at its first step and what is learnt from then
    on; the tensor is its rounding. ``max_norm`` clips the norm over
    all gradients (``grad_norm``, a device tensor, holds the last one); with it a step whose
    norm is not finite changes nothing and does not count. ``seed``: of the 8-bit rounding.

    The step number is the optimiser's, counted from a tensor's first step, the one of its first gradient
    (``before`` in its state holds the steps before); a tensor without a gradient is left as it is. The
    step runs on the current stream and does not synchronise; it cannot be captured into a CUDA
    graph (the step number is the host's)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32,
                 max_norm=None, seed=0):  # fmt: skip
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm must be above 0, not {max_norm}")
        self.state_bits, self.max_norm, self.seed = state_bits, max_norm, int(seed) & 0xFFFFFFFF
        self.steps = 0
        self._control = self._partial = self._batches = None
        super().__init__(params, {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay})

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
        except Exception:
            self.param_groups.pop()
            raise

    def _check_group(self, group):
        (b1, b2), eps = group["betas"], group["eps"]
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be in [0, 1), not {group['betas']}")
        if not (eps > 0.0 or (eps == 0.0 and self.state_bits == 32)):
            raise ValueError(f"eps must be above 0, not {eps}")
        if not (group["lr"] >= 0.0 and group["weight_decay"] >= 0.0):
            raise ValueError(f"lr and weight_decay must not be negative: {group['lr']}, {group['weight_decay']}")
        for p in group["params"]:
            if not p.is_cuda:
                raise RuntimeError("wiretorch_b200 runs on CUDA tensors only (no CPU path)")
            if p.dtype not in TYPES:
                raise TypeError(f"AdamW takes float32, bfloat16 and float16 tensors, not {p.dtype}")
            if not _dense(p):
                raise ValueError(f"a learnt tensor must fill one stretch of memory: strides {p.stride()} of {tuple(p.shape)}")
            if p.device != self._device():
                raise ValueError(f"all learnt tensors must be on one GPU: {p.device} and {self._device()}")

    def _device(self):
        return next(p.device for group in self.param_groups for p in group["params"])

    # --- the norm's result, on the device (WtStepControl) ---

    def _control_of(self, device):
        if self._control is None:
            self._control = torch.zeros(6, dtype=torch.int32, device=device)
        return self._control

    @property
    def grad_norm(self):
        """The last step's gradient norm before clipping, a device tensor (None without max_norm)."""
        return None if self._control is None else self._control[:1].view(torch.float32)[0]

    def _skipped_at(self):
        return self._control[SKIPPED // 4 :].view(torch.int64)

    @property
    def skipped(self) -> int:
        """Steps left out so far (reads the device)."""
        return 0 if self._control is None else int(self._skipped_at())

    # --- state ---

    def _new_state(self, p):
        with torch.no_grad():
            held = {}
            if self.state_bits == 32:
                held["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
                held["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
            else:
                blocks = -(-p.numel() // BLOCK)
                for name in ("exp_avg", "exp_avg_sq"):
                    held[name] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
                    held[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
            if p.dtype != torch.float32:
                held["master"] = p.detach().float()
            if self.steps:
                held["before"] = torch.full((1,), self.steps, dtype=torch.int64, device=p.device)
                if self._control is not None:
                    held["before"] -= self._skipped_at()
        return held

    def _checked_state(self, p):
        held = self.state[p]
        if not held:
            self.state[p] = held = self._new_state(p)
        kind = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        names = [("exp_avg", kind), ("exp_avg_sq", kind)]
        if p.dtype != torch.float32:
            names.append(("master", torch.float32))
        before = held.get("before")
        if before is not None and (before.dtype != torch.int64 or before.numel() != 1 or before.device != p.device):
            raise ValueError("the state's before must be one int64 on its tensor's device")
        for name, want in names:
            t = held[name]
            if t.dtype != want or t.shape != p.shape or t.device != p.device or t.stride() != p.stride():
                raise ValueError(f"the state's {name} must be {want} with its tensor's shape, strides and device")
        if self.state_bits == 8:
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                t = held[name]
                if t.dtype != torch.float32 or t.numel() != -(-p.numel() // BLOCK) or not t.is_contiguous() or t.device != p.device:
                    raise ValueError(f"the state's {name} must be contiguous float32, one per {BLOCK} elements")
        return held

    def _plan(self, with_grad):
        """Batches of the tensors that have a gradient, checked."""
        eight, batches, first = self.state_bits == 8, {}, 0
        for group in self.param_groups:
            self._check_group(group)
            key = (tuple(group["betas"]), group["eps"])
            for p in group["params"]:
                at = first
                first += -(-p.numel() // BLOCK) * BLOCK
                if p in with_grad and p.numel():
                    kind = (p.dtype, *key)
                    if kind not in batches:
                        batches[kind] = _Batch(*kind)
                    batches[kind].add(p, self._checked_state(p), group, at)
        for batch in batches.values():
            names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_scale", "exp_avg_sq_scale"] if eight else [])
            batch.close(names + (["master"] if batch.dtype != torch.float32 else []))
        return list(batches.values())

    def _state_now(self):
        return list(chain.from_iterable(map(dict.values, self.state.values())))

    def _current_batches(self):
        """The batches of the tensors that have a gradient now: the last step's, where nothing but
        gradients and rates changed since, and their gradients, in the order of each tensor's memory."""
        held, groups = self._batches, self.param_groups
        every = params = [p for group in groups for p in group["params"]]
        grads = list(map(_grad, params))
        if not all(map(is_not, grads, repeat(None))):
            params = [p for p, g in zip(params, grads) if g is not None]
            grads = [g for g in grads if g is not None]
        settings = [(tuple(group["betas"]), group["eps"], len(group["params"])) for group in groups]
        if (held is None or held[0] != settings or not _same(held[1], groups) or not _same(held[2], every)
                or not (params is every and held[3] is held[2] or _same(held[3], params))
                or not _same(held[5], self._state_now()) or not all(map(_Batch.is_current, held[4]))):  # fmt: skip
            batches = self._plan(set(params))
            held = self._batches = (settings, list(groups), every, params, batches, self._state_now())
        batches = held[4]
        if len(batches) != 1 or len(batches[0].params) != len(params):
            grads = [list(map(_grad, batch.params)) for batch in batches]
        else:
            grads = [grads]
        for i, batch in enumerate(batches):
            if not batch.takes(grads[i]):
                grads[i] = [self._in_order(p, g) for p, g in zip(batch.params, grads[i])]
        return batches, grads

    @staticmethod
    def _in_order(p, g):
        if g.layout != torch.strided:
            raise TypeError("AdamW takes dense gradients only")
        if g.dtype != p.dtype or g.device != p.device or g.shape != p.shape:
            raise TypeError(f"a gradient must have its tensor's type, shape and device: {g.dtype}, {tuple(g.shape)} on "
                            f"{g.device}; {p.dtype}, {tuple(p.shape)} on {p.device}")  # fmt: skip
        if g.stride() != p.stride():  # the kernel walks memory: the same order in both
            g = torch.empty_strided(p.shape, p.stride(), dtype=g.dtype, device=g.device).copy_(g)
        return g

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # asked before any state is made: what a refused capture recorded never runs
        if torch.cuda.is_current_stream_capturing() and any(
                p.grad is not None for group in self.param_groups for p in group["params"]):  # fmt: skip
            raise RuntimeError("AdamW.step cannot be captured into a CUDA graph: its step number is the host's")
        batches, grads = self._current_batches()
        if not batches:
            return loss
        device = batches[0].params[0].device
        if device.index == torch.cuda.current_device():
            self._run(batches, grads, device)
        else:
            with torch.cuda.device(device):
                self._run(batches, grads, device)
        return loss

    def _run(self, batches, grads, device):
        stream = _C.c_void_p(_lib.stream_of(device))
        at = [_addresses(gs) for gs in grads]
        if self.max_norm is not None:
            self._norm(batches, at, device, stream)
        self.steps += 1
        for batch, g in zip(batches, at):
            self._launch(batch, g, stream)
            torch.autograd.graph.increment_version(batch.params)

    def _norm(self, batches, grads, device, stream):
        lib, a = _lib.lib(), _GradNorm()
        g, numel, kinds = grads[0], batches[0].counts, batches[0].types
        for batch, more in zip(batches[1:], grads[1:]):
            g, numel, kinds = g + more, numel + batch.counts, kinds + batch.types
        n = len(g)
        need = lib.wt_grad_norm_partials(n)
        if self._partial is None or self._partial.numel() < need:
            self._partial = torch.empty(need, dtype=torch.float64, device=device)
        a.n, a.g, a.numel, a.type = n, _at(g), _at(numel), _at(kinds)
        a.max_norm, a.partial = self.max_norm, self._partial.data_ptr()
        a.control = self._control_of(device).data_ptr()
        with _lib.timed("wt_grad_norm"):
            rc = lib.wt_grad_norm(_C.byref(a), stream)
        _lib.check(rc, "wt_grad_norm")
        _lib.count_launches(1)

    def _launch(self, batch, g, stream):
        a = _AdamW()
        p, state = _addresses(batch.params), {name: _addresses(kept) for name, kept in batch.state.items()}
        lr, decay = batch.rates("lr"), batch.rates("weight_decay")
        a.n, a.type, a.state_bits = len(g), TYPES[batch.dtype], self.state_bits
        a.p, a.g, a.m, a.v = _at(p), _at(g), _at(state["exp_avg"]), _at(state["exp_avg_sq"])
        if self.state_bits == 8:
            a.m_scale, a.v_scale = _at(state["exp_avg_scale"]), _at(state["exp_avg_sq_scale"])
        if "master" in state:
            a.master = _at(state["master"])
        a.numel, a.first, a.lr, a.weight_decay = _at(batch.counts), _at(batch.firsts), _at(lr), _at(decay)
        (a.beta1, a.beta2), a.eps = batch.betas, batch.eps
        a.step, a.count, a.seed = self.steps, self.steps, self.seed
        if batch.before is not None:
            before = array("Q", [0 if t is None else t.data_ptr() for t in batch.before])
            a.before = _at(before)
        if self._control is not None:  # what was left out counts on without a limit, too
            at = self._control.data_ptr()
            a.control, a.skipped = None if self.max_norm is None else at, at + SKIPPED
        with _lib.timed("wt_adamw_step"):
            rc = _lib.lib().wt_adamw_step(_C.byref(a), stream)
        _lib.check(rc, "wt_adamw_step")
        _lib.count_launches(1)

    # --- saving ---

    def state_dict(self):
        return super().state_dict() | {"wiretorch": {"state_bits": self.state_bits, "seed": self.seed,
                                                     "steps": self.steps, "skipped": self.skipped}}  # fmt: skip

    def load_state_dict(self, state_dict):
        own = state_dict.get("wiretorch")
        if own is None:
            raise ValueError("not a state of wiretorch_b200.optim.AdamW")
        if own["state_bits"] != self.state_bits:
            raise ValueError(f"the state has {own['state_bits']}-bit moments, this optimiser {self.state_bits}")
        super().load_state_dict({k: v for k, v in state_dict.items() if k != "wiretorch"})
        # torch casts a loaded state to its tensor's type: put the moments back as they were
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                self.state[p] = {k: t.detach().to(p.device, copy=True) for k, t in state_dict["state"][i].items()}
        for group in self.param_groups:  # a state that has the steps before a group was added with the group
            born = group.pop("born", 0)
            for p in group["params"] if born else ():
                if self.state.get(p):
                    self.state[p].setdefault("before", torch.full((1,), born, dtype=torch.int64, device=p.device))
        self._batches = None
        self.steps, self.seed = own["steps"], own["seed"]
        if own["skipped"] or self._control is not None:
            self._control_of(self._device())
            self._skipped_at().fill_(own["skipped"])

    def __getstate__(self):
        own = ("state_bits", "max_norm", "seed", "steps", "_control")
        return super().__getstate__() | {k: getattr(self, k) for k in own}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._partial = self._batches = None
