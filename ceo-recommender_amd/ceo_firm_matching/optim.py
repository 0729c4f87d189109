"""AdamW over many tensors in one launch (HIP kernel ``tt_adamw_step``).

The reference trains with ``optim.Adam`` (training.py:32, contrastive.py:219);
the fused two-tower step applies it over one flat arena (``FusedTrainer``).
This optimizer takes any list of parameters -- ``train_contrastive`` uses it
for towers and projector heads together -- with decoupled weight decay and
states in 32 or in 8 bits.
"""
from __future__ import annotations

import ctypes
from itertools import chain
from operator import attrgetter
from typing import Optional

import numpy as np
import torch

from . import _native as N
from . import block8

# over lists of parameters at every step: called without a Python frame each
_grad, _dtype = attrgetter("grad"), attrgetter("dtype")
_numel, _contiguous, _address = torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.data_ptr


def _likeness(tensors):
    return [list(map(_numel, tensors)), list(map(_dtype, tensors)), list(map(torch.Tensor.get_device, tensors))]


_BYTES = ("exp_avg_codes", "exp_avg_scales", "exp_avg_sqrt_codes", "exp_avg_sqrt_scales")


class _Bucket:
    """The states of one parameter group: arenas of blocks of 128 values, each
    parameter from a block of its own."""

    def __init__(self, params, bits, capturable):
        self.params = params
        self.device = params[0].device if params else torch.device("cpu")
        self.numel = [p.numel() for p in params]
        self.like = _likeness(params)  # what a step has to find
        nb = [block8.blocks_of(n) for n in self.numel]
        self.block0 = [0] * len(nb)
        for i in range(1, len(nb)):
            self.block0[i] = self.block0[i - 1] + nb[i - 1]
        self.nb, self.n_blocks = nb, sum(nb)
        dev = self.device
        if bits == 32:
            self.m = torch.zeros(self.n_blocks, block8.BLOCK, device=dev)
            self.v = torch.zeros(self.n_blocks, block8.BLOCK, device=dev)
            self.arenas = {"exp_avg": self.m, "exp_avg_sq": self.v}
        else:
            self.arenas = {k: (torch.full((self.n_blocks,), 127, dtype=torch.uint8, device=dev) if k.endswith("scales")
                               else torch.zeros(self.n_blocks, block8.BLOCK, dtype=torch.uint8, device=dev))
                           for k in _BYTES}
        self.steps = torch.zeros(len(params), dtype=torch.int64, device=dev if capturable else "cpu")
        self.coefs = torch.zeros(max(1, len(params)), 4, device=dev) if capturable else None
        self.host_steps = None if capturable else self.steps.numpy()
        self.table = np.zeros((len(params), 6), dtype=np.int64)  # tt_adamw_tensor rows
        self.table[:, 2] = self.numel
        self.table[:, 3] = self.block0
        self.table[:, 5] = [N.DTYPES[p.dtype] for p in params]
        self.table_at = self.table.ctypes.data
        s = N.TTAdamWState()
        if dev.type == "cuda":
            for field, t in zip(("exp_avg", "exp_avg_sq") if bits == 32 else ("m_codes", "m_scales", "r_codes", "r_scales"),
                                self.arenas.values()):
                setattr(s, field, t.data_ptr())
            if capturable:
                s.steps, s.coefs, s.n_steps = self.steps.data_ptr(), self.coefs.data_ptr(), len(params)
        s.n_blocks = self.n_blocks
        self.native = s

    def views(self, i):
        """Parameter i's states, shaped like it (scales: one byte a block)."""
        b0, nb, p = self.block0[i], self.nb[i], self.params[i]
        out = {"step": self.steps[i]}
        for k, a in self.arenas.items():
            part = a[b0:b0 + nb]
            out[k] = part if k.endswith("scales") else part.reshape(-1)[:p.numel()].view(p.shape)
        return out


class AdamW(torch.optim.Optimizer):
    """AdamW: ``p -= lr * weight_decay * p``, then Adam's step.

    ``state_bits=32``: ``exp_avg`` and ``exp_avg_sq`` in float32 whatever the
    parameters' type; ``state_dict`` holds them under torch.optim.AdamW's names.
    ``state_bits=8``: ``exp_avg`` in e4m3 and ``sqrt(exp_avg_sq)`` in unsigned
    e4m4, blocks of 128 values with a power-of-two scale: 2.02 bytes a value
    instead of 8.  Both are rounded up or down with the probability of what is
    cut off (nearest would freeze them: a step moves exp_avg_sq by 0.1 %, half a
    step of 8 bits is 3 %), by a hash of ``seed``, the step and the value's place,
    so equal runs stay equal.

    Parameters: float32, bfloat16, float16, contiguous; one device per group.
    Arithmetic in 32 bits, the parameter rounded once.  Parameters without a
    gradient are skipped, their step count too.  ``capturable=True`` keeps the
    step counts on the device so that ``step`` can be captured into a graph
    (the graph keeps the learning rate it was captured with).  CPU parameters
    run the same formulas in torch ops.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32, seed: int = 0, capturable: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, got {state_bits}")
        self._bits, self._seed, self._capturable = int(state_bits), int(seed) & block8.M64, bool(capturable)
        self._buckets = []
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    # -- groups ---------------------------------------------------------------
    @staticmethod
    def _check_hyper(g):
        b1, b2 = g["betas"]
        if not g["lr"] >= 0 or not np.isfinite(g["lr"]):
            raise ValueError(f"Invalid learning rate: {g['lr']}")
        if not 0 <= b1 < 1 or not 0 <= b2 < 1:
            raise ValueError(f"Invalid betas: {g['betas']}")
        if not g["eps"] >= 0 or not np.isfinite(g["eps"]):
            raise ValueError(f"Invalid epsilon value: {g['eps']}")
        if not g["weight_decay"] >= 0 or not np.isfinite(g["weight_decay"]):
            raise ValueError(f"Invalid weight_decay value: {g['weight_decay']}")

    @staticmethod
    def _check_options(g):
        """Options of torch's optimizers under which its step is another one."""
        for option in ("maximize", "amsgrad", "differentiable"):
            if g.get(option):
                raise NotImplementedError(f"AdamW: {option}={g[option]} is not supported")
        if not g.get("decoupled_weight_decay", True) and g["weight_decay"] != 0:
            raise NotImplementedError("AdamW: weight decay that is added to the gradient is not supported")

    @staticmethod
    def _check_apart(params):
        """One launch updates all of them: no value may be in two."""
        at = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
        if any(a[1] > b[0] for a, b in zip(at, at[1:])):
            raise ValueError("AdamW: parameters of a group share memory (the same parameter twice, or overlapping views)")

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        g = self.param_groups[-1]
        try:
            self._check_hyper(g)
            self._check_options(g)
            for p in g["params"]:
                if p.dtype not in N.DTYPES:
                    raise NotImplementedError(f"AdamW: float32, bfloat16 or float16 parameters, got {p.dtype}")
                if p.layout != torch.strided or not p.is_contiguous():
                    raise ValueError("AdamW: parameters must be contiguous")
                if p.device != g["params"][0].device:
                    raise ValueError("AdamW: one device per parameter group")
                if p.device.type not in ("cuda", "cpu"):
                    raise NotImplementedError(f"AdamW: HIP or CPU parameters, got {p.device}")
            self._check_apart(g["params"])
            if self._capturable and g["params"] and g["params"][0].device.type != "cuda":
                raise ValueError("AdamW: capturable needs parameters on a HIP device")
        except Exception:
            self.param_groups.pop()
            raise
        self._bind(g)

    def _bind(self, g):
        b = _Bucket(g["params"], self._bits, self._capturable)
        self._buckets.append(b)
        for i, p in enumerate(b.params):
            self.state[p] = b.views(i)

    # -- one step -------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        steps = []  # every group is checked before the first one steps
        for g, b in zip(self.param_groups, self._buckets):
            live, params, grads = None, b.params, list(map(_grad, b.params))
            try:
                dense = list(map(_contiguous, grads))
            except TypeError:  # parameters without a gradient among them
                live = [i for i, x in enumerate(grads) if x is not None]
                params, grads = [params[i] for i in live], [grads[i] for i in live]
                dense = [x.layout == torch.strided and x.is_contiguous() for x in grads]
            except RuntimeError:
                dense = [False]
            if not params:
                continue
            like = b.like if live is None else [[x[i] for i in live] for x in b.like]
            if _likeness(params) != like or not all(map(_contiguous, params)):
                raise RuntimeError("AdamW: a parameter changed its size, type, device or layout after the optimizer was made")
            if _likeness(grads) != like:
                raise RuntimeError("AdamW: a gradient's size, type or device is not its parameter's")
            if not all(dense):
                if any(x.layout != torch.strided for x in grads):
                    raise NotImplementedError("AdamW: sparse gradients are not supported")
                grads = [x.contiguous() for x in grads]
            if b.device.type != "cuda" or len(self._buckets) > 1:  # (a single HIP group's step checks them itself)
                self._check_hyper(g)
                if b.device.type == "cuda":
                    with N.on_device(b.device):
                        self._check_capture()
            steps.append((g, b, live, params, grads))
        for g, b, live, params, grads in steps:
            if b.device.type == "cuda":
                self._step_hip(g, b, live, params, grads)
            else:
                self._step_cpu(g, b, range(len(params)) if live is None else live, grads)
        return loss

    def _check_capture(self):
        if not self._capturable and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a captured step needs capturable=True (the step count would be frozen)")

    def _step_hip(self, g, b, live, params, grads):
        with N.on_device(b.device):
            self._check_capture()
            t, at = (b.table, b.table_at) if live is None else (b.table[live], 0)
            t[:, 0] = list(map(_address, params))
            t[:, 1] = list(map(_address, grads))
            if self._capturable:
                t[:, 4] = range(len(params)) if live is None else live
            else:
                t[:, 4] = (b.host_steps if live is None else b.host_steps[live]) + 1
            hp = N.TTAdamWHP(g["lr"], g["betas"][0], g["betas"][1], g["eps"], g["weight_decay"])
            N.check(N.lib().tt_adamw_step(at or t.ctypes.data, len(params), self._bits, ctypes.byref(b.native),
                                          ctypes.byref(hp), self._seed, N.stream_ptr(b.device)), "tt_adamw_step")
            if not self._capturable:  # the step was taken
                b.host_steps[slice(None) if live is None else live] = t[:, 4]
        torch.autograd.graph.increment_version(params)

    def _step_cpu(self, g, b, live, grads):
        b1, b2 = g["betas"]
        for i, gr in zip(live, grads):
            b.host_steps[i] += 1
            t, p = int(b.host_steps[i]), b.params[i]
            n, at = p.numel(), slice(b.block0[i], b.block0[i] + b.nb[i])
            if n == 0:
                continue
            pad = lambda x: torch.nn.functional.pad(x.reshape(-1).to(torch.float32),  # noqa: E731
                                                    (0, -n % block8.BLOCK)).reshape(-1, block8.BLOCK)
            x, gf = pad(p), pad(gr)
            if self._bits == 32:
                m, v = b.m[at], b.v[at]
            else:
                mc, ms, rc, rs = (b.arenas[k][at] for k in _BYTES)
                m = block8.held(mc, ms, block8.E4M3)
                v = block8.held(rc, rs, block8.E4M4).square()
            m = gf - b1 * (gf - m) if b1 < 0.5 else m + (1 - b1) * (gf - m)
            v = b2 * v + (1 - b2) * gf * gf
            r = v.sqrt()
            x = x * (1 - g["lr"] * g["weight_decay"]) - (g["lr"] / (1 - b1 ** t)) * (m / (r / (1 - b2 ** t) ** 0.5 + g["eps"]))
            p.copy_(x.reshape(-1)[:n].view(p.shape))
            if self._bits == 32:
                b.m[at], b.v[at] = m, v
            else:
                um, ur = block8.rounding_bits(b.block0[i], b.nb[i], self._seed, t)
                mc[:], ms[:] = block8.hold(m, um, block8.E4M3, False)
                rc[:], rs[:] = block8.hold(r, ur, block8.E4M4, True)
                if n % block8.BLOCK:  # the padding stays zero
                    mc[-1, n % block8.BLOCK:] = 0
                    rc[-1, n % block8.BLOCK:] = 0

    # -- states ---------------------------------------------------------------
    def held_states(self, group: int = 0):
        """What the optimizer holds for a parameter group, as arenas [blocks,
        128] in which every parameter starts a new block: ``(exp_avg,
        exp_avg_sq)`` themselves in 32 bits; with 8-bit states the values of
        ``(exp_avg, sqrt(exp_avg_sq))`` in bfloat16, which holds them exactly."""
        b = self._buckets[group]
        if self._bits == 32:
            return b.m, b.v
        mc, ms, rc, rs = (b.arenas[k] for k in _BYTES)
        if b.device.type != "cuda":
            return (block8.held(mc, ms, block8.E4M3).to(torch.bfloat16),
                    block8.held(rc, rs, block8.E4M4).to(torch.bfloat16))
        with N.on_device(b.device):
            m = torch.empty(b.n_blocks, block8.BLOCK, dtype=torch.bfloat16, device=b.device)
            r = torch.empty_like(m)
            N.check(N.lib().tt_adamw_held(ctypes.byref(b.native), m.data_ptr(), r.data_ptr(), N.stream_ptr(b.device)),
                    "tt_adamw_held")
        return m, r

    def load_state_dict(self, state_dict):
        """Hyperparameters and states, copied into the arenas that the steps
        (captured ones too) already use.  8-bit states load from 8-bit ones
        only; 32-bit ones also from ``torch.optim.AdamW``'s.  Options that
        this step does not follow (``maximize``, ``amsgrad``,
        ``differentiable``, a decay that is not decoupled) are refused, and
        nothing has changed then."""
        given = state_dict["state"]
        groups = []
        for g in state_dict["param_groups"]:
            g = dict(g)
            g.update({k: float(g[k]) for k in ("lr", "eps", "weight_decay")}, betas=tuple(map(float, g["betas"])))  # (tensors too)
            self._check_hyper(g)
            self._check_options(g)
            g.pop("decoupled_weight_decay", None)
            groups.append(g)
        ids = list(chain.from_iterable(g["params"] for g in groups))
        mine = list(chain.from_iterable(g["params"] for g in self.param_groups))
        if len(ids) == len(mine):  # (another count is the base class's error)
            for k, p in zip(ids, mine):
                for name, a in given.get(k, {}).items():
                    to = self.state[p].get(name)
                    if to is None:
                        raise ValueError(f"AdamW: state {name!r} does not belong to {self._bits}-bit states")
                    if name != "step" and (tuple(a.shape) != tuple(to.shape) or
                                           (to.dtype == torch.uint8) != (a.dtype == torch.uint8)):
                        raise ValueError(f"AdamW: state {name!r} is {tuple(a.shape)} {a.dtype}, "
                                         f"expected {tuple(to.shape)} {to.dtype}")
        keep = self.state
        super().load_state_dict({"state": {}, "param_groups": groups})
        self.state = keep
        with torch.no_grad():
            for k, p in zip(ids, mine):
                st = given.get(k)
                for name, to in self.state[p].items():
                    if st is None or name not in st:
                        to.fill_(127) if name.endswith("scales") else to.zero_()
                    elif name == "step":
                        to.fill_(int(st["step"]))
                    else:
                        to.copy_(st[name])

    def __getstate__(self):
        return {**super().__getstate__(), "_config": (self._bits, self._seed, self._capturable)}

    def __setstate__(self, state):
        config = state.pop("_config", None) if "_config" in state else None
        super().__setstate__(state)
        if config is not None:  # unpickled or deep-copied: arenas of its own again
            self._bits, self._seed, self._capturable = config
            self._buckets, old = [], dict(self.state)
            for g in self.param_groups:
                self._bind(g)
                for p in g["params"]:
                    for name, to in self.state[p].items():
                        to.copy_(old[p][name])
