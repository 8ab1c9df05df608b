"""Optimizers: `Optimizer`, `Adam`, `adam_fused_scalars`
(ttrl/engine/optim/{base,adam,scalars,checkpoint}.py), and `AdamW`, with
decoupled weight decay and moments in 32 or 8 bits.

Adam keeps the reference's stored S = m/(1-b1), V = v/(1-b2) moments and
its per-parameter step counts, and runs as ONE multi-tensor CUDA kernel per
step. The step counts live on the device (the kernel reads and advances
them), so the whole update -- Adam included -- can be captured into a CUDA
graph and replayed with the correct bias correction every time. A host
mirror of the counts backs `state_dict`.
"""

from __future__ import annotations

import math
import operator
from array import array
from itertools import chain

import numpy as np
import torch

from ttrl_b200 import _lib
from ttrl_b200.device import context
from ttrl_b200.engine.tensor import MASTER_DTYPE, restore_in_place, to_host

__all__ = ["Optimizer", "Adam", "AdamW", "adam_bias_table", "adam_fused_scalars", "share_launch",
           "step_together"]


def adam_fused_scalars(lr: float, b1: float, b2: float, eps: float, t: int) -> tuple[float, float]:
    """(alpha_t, eps_t) folding the bias correction (ttrl/engine/optim/scalars.py:13-27)."""
    if t < 1:
        raise ValueError(f"adam_fused_scalars: t must be >= 1, got {t}")
    bc1 = 1 - b1 ** t
    bc2 = 1 - b2 ** t
    c = math.sqrt((1 - b2) / bc2)
    return lr * (1 - b1) / bc1 / c, eps / c


#: Longest bias-term table built (steps); betas that converge later fall
#: back to the kernel's own pow().
BIAS_TABLE_MAX_STEPS = 1 << 20

#: AdamW's smallest eps: the smallest normal float32.
EPS_MIN = 2.0 ** -126

_BIAS_TABLES: dict = {}


def adam_bias_table(b1: float, b2: float, device):
    """(T, 2) float64 device table of (1 - b1^t, sqrt((1 - b2)/(1 - b2^t)))
    for t = 1..T, the terms of adam_fused_scalars from the host's pow(); T
    is the first step at which both have converged to 1 (in double), so the
    kernel reads the last row for every later step. None when that takes
    more than BIAS_TABLE_MAX_STEPS steps. One table per (betas, device)."""
    key = (float(b1), float(b2), str(device))
    if key in _BIAS_TABLES:
        return _BIAS_TABLES[key]
    tiny = math.ldexp(1.0, -54)  # 1 - x == 1 in double once x < 2^-54
    need = 1
    for b in (b1, b2):
        if b > 0.0:
            need = max(need, int(math.ceil(math.log(tiny) / math.log(b))) + 2)
    table = None
    if need <= BIAS_TABLE_MAX_STEPS:
        # Python's own pow (the reference's `b ** t`), not a vectorised one
        # that may round differently.
        rows = []
        for t in range(1, need + 1):
            bc1, bc2 = 1 - b1 ** t, 1 - b2 ** t
            rows.append((bc1, math.sqrt((1 - b2) / bc2)))
            if bc1 == 1.0 and bc2 == 1.0:
                table = torch.tensor(rows, dtype=torch.float64).to(device)
                break
    _BIAS_TABLES[key] = table
    return table


class Optimizer:
    def __init__(self, params):
        self.params = list(params)

    def zero_grad(self) -> None:
        for p in self.params:
            p.zero_grad()

    def step(self) -> None:
        raise NotImplementedError


class Adam(Optimizer):
    """Adam over fp32 parameters, updated in place by one fused kernel."""

    def __init__(self, params, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0):
        super().__init__(params)
        if not self.params:
            raise ValueError("Adam: params is empty, so there is nothing to optimize")
        if lr <= 0:
            raise ValueError(f"Adam: lr must be > 0, got {lr}")
        b1, b2 = betas
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"Adam: betas must be in [0, 1), got {betas}")
        if eps <= 0:
            raise ValueError(f"Adam: eps must be > 0, got {eps}")
        if weight_decay < 0:
            raise ValueError(f"Adam: weight_decay must be >= 0, got {weight_decay}")
        wrong = [i for i, p in enumerate(self.params) if p.data.dtype != MASTER_DTYPE]
        if wrong:
            raise ValueError(f"Adam: parameters must be {MASTER_DTYPE}; parameters {wrong} are not")
        self.b1, self.b2 = b1, b2
        self.eps = eps
        self.weight_decay = weight_decay
        self.t = 0
        self.steps = [0] * len(self.params)
        dev = self.params[0].data.device
        self._device = dev
        self.m = [torch.zeros_like(p.data) for p in self.params]   # S
        self.v = [torch.zeros_like(p.data) for p in self.params]   # V
        self._dev_steps = torch.zeros(len(self.params), dtype=torch.int32, device=dev)
        self._ticket = torch.zeros(1, dtype=torch.int32, device=dev)
        self._lr_dev = torch.zeros(1, dtype=torch.float64, device=dev)
        self._lr = float(lr)
        self._lr_dev.copy_(torch.tensor([self._lr], dtype=torch.float64))
        # Set by a device-side gradient clip for the next step() (see
        # ttrl_b200.algos.grads.clip_grad_norm_device).
        self.grad_scale = None
        # Indices stepped by the launch recorded inside a graph capture.
        self.captured_indices: list[int] | None = None
        # (group, counter base, rate slot) once share_launch joined it.
        self._shared = None
        self._bias = adam_bias_table(b1, b2, dev)

    # The learning rate lives on the device too, so a replayed graph reads
    # the current value (PPO's annealing, ttrl/algos/ppo/learn.py:54-56).
    @property
    def lr(self) -> float:
        return self._lr

    @lr.setter
    def lr(self, value: float) -> None:
        self._lr = float(value)
        self._lr_dev.copy_(torch.tensor([self._lr], dtype=torch.float64))

    @property
    def state_tensors(self) -> list:
        """The device tensors that hold the moments."""
        return self.m + self.v

    @property
    def _m_scale(self) -> float:
        return 1 - self.b1

    @property
    def _v_scale(self) -> float:
        return 1 - self.b2

    def _pending(self, step_base: int = 0, lr_index: int = 0):
        """(tensors, stepped indices) of the parameters that hold a gradient."""
        tensors = []
        stepped = []
        for i, p in enumerate(self.params):
            if p.grad is None:
                continue
            g = p.grad if p.grad.is_contiguous() else p.grad.contiguous()
            tensors.append((p.data, g.reshape(p.data.shape), self.m[i], self.v[i],
                            step_base + i, lr_index))
            stepped.append(i)
        return tensors, stepped

    def _finish(self, stepped) -> None:
        self.grad_scale = None
        if torch.cuda.is_current_stream_capturing():
            # Recorded, not run: TrainStep advances the host mirror per replay.
            self.captured_indices = stepped
            return
        self.advance(stepped)

    def step(self) -> None:
        """One update of every parameter that holds a gradient."""
        tensors, stepped = self._pending()
        if tensors:
            context(self._device).adam_step(
                tensors, self._dev_steps, self._ticket, self.grad_scale, self._lr, self.b1,
                self.b2, self.eps, self.weight_decay, lr_device=self._lr_dev, bias=self._bias)
        self._finish(stepped)

    def advance(self, stepped) -> None:
        """Advance the host mirror of the device step counters."""
        self.t += 1
        for i in stepped:
            self.steps[i] += 1

    def _step_scalars(self, t: int) -> tuple[float, float]:
        return adam_fused_scalars(self._lr, self.b1, self.b2, self.eps, t)

    # -- checkpoint (ttrl/engine/optim/checkpoint.py) ---------------------

    def state_dict(self) -> dict:
        return {
            "t": self.t,
            "steps": list(self.steps),
            "lr": self._lr,
            "betas": (self.b1, self.b2),
            "eps": self.eps,
            "weight_decay": self.weight_decay,
            "m": [self._portable(i, to_host(m) * self._m_scale) for i, m in enumerate(self.m)],
            "v": [self._portable(i, to_host(v) * self._v_scale) for i, v in enumerate(self.v)],
        }

    def _portable(self, i: int, array: np.ndarray) -> np.ndarray:
        """A moment in its parameter's portable layout (a convolution weight's
        in OIHW, every other parameter's as stored)."""
        layout = getattr(self.params[i], "_layout", None)
        return array if layout is None else layout.to_portable(array)

    def load_state_dict(self, state: dict, device=None) -> None:
        if len(state["m"]) != len(self.m) or len(state["v"]) != len(self.v):
            raise ValueError(
                f"Adam.load_state_dict: checkpoint has {len(state['m'])} m and "
                f"{len(state['v'])} v buffers, expected {len(self.m)} of each."
            )
        device_form = {"m": [], "v": []}
        for key, buffers in (("m", self.m), ("v", self.v)):
            for i, (arr, buf) in enumerate(zip(state[key], buffers)):
                layout = getattr(self.params[i], "_layout", None)
                got = tuple(np.asarray(arr).shape)
                if layout is not None:
                    # Logical OIHW or the reference's prepared matrix; the
                    # stored v fixes the latter's channel stride.
                    try:
                        arr = layout.from_stored(arr, v=state["v"][i])
                    except ValueError as exc:
                        raise ValueError(
                            f"Adam.load_state_dict: {key}[{i}] has shape {got}, which is "
                            f"neither its convolution weight's OIHW shape {layout.oihw} nor "
                            f"a prepared matrix holding it ({exc})") from None
                elif got != tuple(buf.shape):
                    raise ValueError(
                        f"Adam.load_state_dict: {key}[{i}] has shape {got}, which does "
                        f"not match its parameter's shape {tuple(buf.shape)}."
                    )
                device_form[key].append(arr)
        t = int(state["t"])
        steps = [int(s) for s in state.get("steps", [t] * len(self.params))]
        lr = state.get("lr", self._lr)
        b1, b2 = state.get("betas", (self.b1, self.b2))
        eps = state.get("eps", self.eps)
        weight_decay = state.get("weight_decay", self.weight_decay)
        if len(steps) != len(self.params):
            raise ValueError(f"Adam.load_state_dict: checkpoint has {len(steps)} step counters, "
                             f"expected {len(self.params)}.")
        if t < 0 or any(s < 0 for s in steps):
            raise ValueError(f"Adam.load_state_dict: step counts must be >= 0, got t={t}.")
        if not lr > 0:
            raise ValueError(f"Adam.load_state_dict: lr must be > 0, got {lr}.")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"Adam.load_state_dict: betas must be in [0, 1), got {(b1, b2)}.")
        if not eps > 0:
            raise ValueError(f"Adam.load_state_dict: eps must be > 0, got {eps}.")
        if weight_decay < 0:
            raise ValueError(f"Adam.load_state_dict: weight_decay must be >= 0, got {weight_decay}.")
        self.t = t
        self.steps = steps
        self.lr = lr
        self.b1, self.b2 = b1, b2
        self.eps = eps
        self.weight_decay = weight_decay
        self._bias = adam_bias_table(self.b1, self.b2, self._device)
        ms, vs = self._m_scale, self._v_scale
        for i, arr in enumerate(device_form["m"]):
            restore_in_place(self.m[i], np.asarray(arr) / ms)
        for i, arr in enumerate(device_form["v"]):
            restore_in_place(self.v[i], np.asarray(arr) / vs)
        self._dev_steps.copy_(torch.tensor(steps, dtype=torch.int32))


class _SharedLaunch:
    """Device state that several Adams keep side by side so that one kernel
    launch can step them all: their step counters in one int32 array, their
    learning rates in one float64 array, one ticket."""

    def __init__(self, opts):
        dev = opts[0]._device
        counts = [len(o.params) for o in opts]
        self.steps = torch.zeros(sum(counts), dtype=torch.int32, device=dev)
        self.lrs = torch.zeros(len(opts), dtype=torch.float64, device=dev)
        self.ticket = torch.zeros(1, dtype=torch.int32, device=dev)
        self.opts = list(opts)
        self.bases = []
        base = 0
        for slot, (o, n) in enumerate(zip(opts, counts)):
            self.steps[base:base + n].copy_(o._dev_steps)
            self.lrs[slot:slot + 1].copy_(o._lr_dev)
            # Views: every in-place write of the optimizer (load_state_dict,
            # the lr setter, a restore) lands in the shared arrays.
            o._dev_steps = self.steps[base:base + n]
            o._lr_dev = self.lrs[slot:slot + 1]
            o._shared = (self, base, slot)
            self.bases.append(base)
            base += n


def share_launch(opts) -> None:
    """Let `step_together(opts)` step these Adams in one kernel launch. Each
    keeps its own parameters, moments, step counters, learning rate and
    state_dict; only where the device copies of the counters and the rate
    live changes. All must be on one device."""
    opts = list(opts)
    if len(opts) < 2:
        return
    if any(not isinstance(o, Adam) for o in opts):
        raise TypeError("share_launch: Adam optimizers only")
    if len({o._device for o in opts}) != 1:
        raise ValueError("share_launch: the optimizers live on different devices")
    if sum(len(o.params) for o in opts) > 64:
        raise ValueError("share_launch: more than 64 parameters in all")
    _SharedLaunch(opts)


def step_together(opts) -> None:
    """step() every optimizer of `opts`: one launch when they were joined by
    share_launch and agree on betas, eps and weight decay with no gradient
    scale pending (the math per parameter is unchanged: each reads its own
    counter and rate); otherwise one step() each, in order."""
    opts = list(opts)
    shared = [getattr(o, "_shared", None) for o in opts]
    group = shared[0][0] if shared and shared[0] is not None else None
    joint = (group is not None and all(s is not None and s[0] is group for s in shared)
             and all(o.grad_scale is None for o in opts)
             and len({(o.b1, o.b2, o.eps, o.weight_decay) for o in opts}) == 1
             and len({id(o._bias) for o in opts}) == 1)
    if not joint:
        for o in opts:
            o.step()
        return
    tensors, stepped = [], []
    for o, (_, base, slot) in zip(opts, shared):
        t, s = o._pending(base, slot)
        tensors += t
        stepped.append(s)
    if tensors:
        head = opts[0]
        context(head._device).adam_step(tensors, group.steps, group.ticket, None, head._lr,
                                        head.b1, head.b2, head.eps, head.weight_decay,
                                        lr_device=group.lrs, bias=head._bias)
    for o, s in zip(opts, stepped):
        o._finish(s)



def _spread(sizes, align: int):
    """(offsets, total) of buffers laid end to end on multiples of `align`."""
    offsets, total = [], 0
    for n in sizes:
        offsets.append(total)
        total += (n + align - 1) // align * align
    return offsets, total


class AdamW(Optimizer):
    """AdamW over fp32 parameters, any number of them, updated in place by
    one kernel launch for every 384: the decay shrinks the parameter itself,
    p (1 - lr wd), where Adam adds it to the gradient.

    `state_bits` 8 keeps both moments of every parameter of at least
    `min_8bit_size` elements as 8-bit codes in blocks of 256 that share a
    scale (shorter ones stay in 32 bits): 2.03 bytes an element instead of 8.
    The parameters and the step's arithmetic stay in 32 bits.

    Steps inside a captured graph, follows `lr` from replay to replay, takes
    the factor of `clip_grad_norm_device`, and reads and writes the same
    `state_dict` as Adam (canonical m and v), so either optimizer and either
    width of state resumes from the other's. A parameter of zero elements is
    left alone. No reference counterpart."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *,
                 state_bits: int = 32, min_8bit_size: int = 4096):
        super().__init__(params)
        if not self.params:
            raise ValueError("AdamW: params is empty, so there is nothing to optimize")
        if not lr > 0:
            raise ValueError(f"AdamW: lr must be > 0, got {lr}")
        b1, b2 = betas
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {betas}")
        if not eps >= EPS_MIN:
            raise ValueError(f"AdamW: eps must be at least 2^-126 (the step divides in float32), "
                             f"got {eps}")
        if not weight_decay >= 0:
            raise ValueError(f"AdamW: weight_decay must be >= 0, got {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {state_bits}")
        if min_8bit_size < 1:
            raise ValueError(f"AdamW: min_8bit_size must be >= 1, got {min_8bit_size}")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("AdamW: a parameter is listed twice")
        wrong = [i for i, p in enumerate(self.params) if p.data.dtype != MASTER_DTYPE]
        if wrong:
            raise ValueError(f"AdamW: parameters must be {MASTER_DTYPE}; parameters {wrong} "
                             "are not")
        dev = self.params[0].data.device
        if any(p.data.device != dev for p in self.params):
            raise ValueError("AdamW: the parameters live on different devices")
        if dev.type != "cuda":
            raise ValueError(f"AdamW runs on CUDA devices only, got parameters on {dev}")
        self._device = dev
        self._keep_apart([p.data for p in self.params])
        self.b1, self.b2 = float(b1), float(b2)
        self.eps = float(eps)
        self.weight_decay = float(weight_decay)
        self.state_bits = int(state_bits)
        self.t = 0
        self.steps = [0] * len(self.params)
        self._numels = [int(p.data.numel()) for p in self.params]
        #: Bits each parameter's moments are held in.
        self.bits = [8 if state_bits == 8 and n >= min_8bit_size else 32 for n in self._numels]
        # The 32-bit moments lie in two flat buffers, each parameter's at a
        # 256-byte boundary in order; the codes and scales in four.
        full = [n if b == 32 else 0 for n, b in zip(self._numels, self.bits)]
        offsets, total = _spread(full, 64)
        self._m32 = torch.zeros(total, device=dev)
        self._v32 = torch.zeros(total, device=dev)
        short = [n if b == 8 else 0 for n, b in zip(self._numels, self.bits)]
        code_at, codes = _spread(short, _lib.ADAMW_BLOCK)
        self._m8 = torch.zeros(codes, dtype=torch.int8, device=dev)
        self._v8 = torch.zeros(codes, dtype=torch.uint8, device=dev)
        self._m_scale = torch.zeros(codes // _lib.ADAMW_BLOCK, device=dev)
        self._v_scale = torch.zeros(codes // _lib.ADAMW_BLOCK, device=dev)
        #: Each parameter's moments: fp32 in its shape, or its codes, flat.
        self.m, self.v = [], []
        table = np.zeros(len(self.params), _lib.ADAMW_TENSOR)
        for i, p in enumerate(self.params):
            n = self._numels[i]
            if self.bits[i] == 32:
                self.m.append(self._m32[offsets[i]:offsets[i] + n].reshape(p.data.shape))
                self.v.append(self._v32[offsets[i]:offsets[i] + n].reshape(p.data.shape))
            else:
                self.m.append(self._m8[code_at[i]:code_at[i] + n])
                self.v.append(self._v8[code_at[i]:code_at[i] + n])
                block = code_at[i] // _lib.ADAMW_BLOCK
                table["m_scale"][i] = self._m_scale[block:].data_ptr()
                table["v_scale"][i] = self._v_scale[block:].data_ptr()
            table["m"][i] = self.m[i].data_ptr()
            table["v"][i] = self.v[i].data_ptr()
        table["numel"] = self._numels
        table["step_index"] = np.arange(len(self.params))
        table["bits"] = self.bits
        self._table = table
        self._dev_steps = torch.zeros(len(self.params), dtype=torch.int32, device=dev)
        self._ticket = torch.zeros(1, dtype=torch.int32, device=dev)
        self._lr = float(lr)
        self._lr_dev = torch.full((1,), self._lr, dtype=torch.float64, device=dev)
        self.grad_scale = None
        self.captured_indices: list[int] | None = None
        self._seen: list = []
        self._seen_at = np.zeros(0, np.uint64)
        self._all = list(range(len(self.params)))
        self._any_empty = not all(self._numels)
        self._bias = adam_bias_table(self.b1, self.b2, dev)

    @property
    def lr(self) -> float:
        return self._lr

    @lr.setter
    def lr(self, value: float) -> None:
        self._lr = float(value)
        self._lr_dev.copy_(torch.tensor([self._lr], dtype=torch.float64))

    @property
    def state_tensors(self) -> list:
        """The device tensors that hold the moments: values, codes, scales."""
        return [self._m32, self._v32, self._m8, self._v8, self._m_scale, self._v_scale]

    @property
    def moment_arenas(self):
        """The two flat buffers of the 32-bit moments: each parameter's at a
        256-byte boundary, in order, zeros between."""
        return self._m32, self._v32

    def step(self) -> None:
        """One update of every parameter that holds a gradient."""
        datas = [p.data for p in self.params]
        grads = [p.grad for p in self.params]
        stepped, numels = self._all, self._numels
        if self._any_empty or any(g is None for g in grads):
            stepped = [i for i, g in enumerate(grads) if g is not None and self._numels[i]]
            datas, grads = [datas[i] for i in stepped], [grads[i] for i in stepped]
            numels = [self._numels[i] for i in stepped]
        if not all(map(torch.Tensor.is_contiguous, grads)):
            grads = [g.contiguous() for g in grads]  # held until the launch is issued
        self._look_over("gradient", grads, numels, stepped)
        at = np.frombuffer(array("Q", map(torch.Tensor.data_ptr, chain(datas, grads))),
                           np.uint64)
        where = at[:len(datas)]
        # The parameters are looked over again when one has been rebound, moved
        # or resized.
        if (len(datas) != len(self._seen) or not all(map(operator.is_, datas, self._seen))
                or not np.array_equal(where, self._seen_at)
                or list(map(torch.Tensor.numel, datas)) != numels):
            self._look_over("data", datas, numels, stepped)
            self._keep_apart(datas)
            self._seen, self._seen_at = datas, where
        if not all(map(torch.Tensor.is_contiguous, datas)):
            raise ValueError("AdamW: a parameter has become a strided view")
        if stepped:
            table = self._table
            if len(stepped) < len(table):
                table = table[stepped]
            table["param"], table["grad"] = where, at[len(datas):]
            context(self._device).adamw_step(
                table, self._dev_steps, self._ticket, self.grad_scale, self._lr, self.b1,
                self.b2, self.eps, self.weight_decay, lr_device=self._lr_dev, bias=self._bias)
        self.grad_scale = None
        if torch.cuda.is_current_stream_capturing():
            # Recorded, not run: TrainStep advances the host mirror per replay.
            self.captured_indices = stepped
            return
        self.advance(stepped)

    def _look_over(self, what: str, tensors, numels, at) -> None:
        """Refuse tensors that are not float32 of these sizes on the device."""
        if (list(map(torch.Tensor.numel, tensors)) == numels
                and set(map(torch.Tensor.get_device, tensors)) <= {self._device.index}
                and [x.dtype for x in tensors].count(MASTER_DTYPE) == len(tensors)):
            return
        for i, n, x in zip(at, numels, tensors):
            if x.numel() != n or x.device != self._device or x.dtype != MASTER_DTYPE:
                raise ValueError(f"AdamW: the {what} of parameter {i} is {tuple(x.shape)} "
                                 f"{x.dtype} on {x.device}, expected {n} elements of "
                                 f"{MASTER_DTYPE} on {self._device}")

    @staticmethod
    def _keep_apart(datas) -> None:
        """Refuse parameters that share memory: both updates would race."""
        spans = sorted((x.data_ptr(), x.numel() * x.element_size()) for x in datas if x.numel())
        if any(at + size > after for (at, size), (after, _) in zip(spans, spans[1:])):
            raise ValueError("AdamW: two parameters share memory")

    def advance(self, stepped) -> None:
        """Advance the host mirror of the device step counters."""
        self.t += 1
        if stepped is self._all:
            self.steps = [s + 1 for s in self.steps]
            return
        for i in stepped:
            self.steps[i] += 1

    # -- moments in fp32 ---------------------------------------------------

    def _moments(self, m, v, pack: bool) -> None:
        m, v = list(m), list(v)
        if len(m) != len(self.params) or len(v) != len(self.params):
            raise ValueError(f"AdamW: {len(m)} m and {len(v)} v tensors for "
                             f"{len(self.params)} parameters")
        rows, at, copies = [], [], []
        for i, pair in enumerate(zip(m, v)):
            for t in pair:
                if (t.dtype != torch.float32 or not t.is_contiguous()
                        or t.numel() != self._numels[i] or t.device != self._device):
                    raise ValueError(f"AdamW: moments of parameter {i} must be contiguous "
                                     f"float32 with {self._numels[i]} elements on "
                                     f"{self._device}")
            if self._numels[i] == 0:
                continue
            if self.bits[i] == 32:
                for held, t in zip((self.m[i], self.v[i]), pair):
                    copies.append((held, t) if pack else (t, held))
            else:
                rows.append((pair[0].data_ptr(), pair[1].data_ptr()))
                at.append(i)
        if copies:
            context(self._device).blend(copies)
        if rows:
            table = np.zeros(len(rows), _lib.ADAMW_STATE)
            table["m32"], table["v32"] = [r[0] for r in rows], [r[1] for r in rows]
            own = self._table[at]
            table["m8"], table["v8"], table["numel"] = own["m"], own["v"], own["numel"]
            table["m_scale"], table["v_scale"] = own["m_scale"], own["v_scale"]
            context(self._device).adamw_state_convert(table, pack)

    def read_moments(self, m, v) -> None:
        """The canonical moments into device tensors of the parameters' sizes."""
        self._moments(m, v, False)

    def load_moments(self, m, v, *, t: int) -> None:
        """Set the canonical moments (device tensors of the parameters' sizes)
        and every step counter to t."""
        if t < 0:
            raise ValueError(f"AdamW: step counts must be >= 0, got t={t}")
        self._moments(m, v, True)
        self._set_steps(t, [int(t)] * len(self.params))

    def _set_steps(self, t: int, steps) -> None:
        self.t = int(t)
        self.steps = [int(s) for s in steps]
        self._dev_steps.copy_(torch.tensor(self.steps, dtype=torch.int32))

    # -- checkpoint (the format of ttrl/engine/optim/checkpoint.py) ---------

    def state_dict(self) -> dict:
        m = [torch.empty(n, device=self._device) for n in self._numels]
        v = [torch.empty(n, device=self._device) for n in self._numels]
        self.read_moments(m, v)

        def portable(i, x):
            x = to_host(x).reshape(tuple(self.params[i].data.shape))
            layout = getattr(self.params[i], "_layout", None)
            return x if layout is None else layout.to_portable(x)

        return {
            "t": self.t,
            "steps": list(self.steps),
            "lr": self._lr,
            "betas": (self.b1, self.b2),
            "eps": self.eps,
            "weight_decay": self.weight_decay,
            "m": [portable(i, x) for i, x in enumerate(m)],
            "v": [portable(i, x) for i, x in enumerate(v)],
        }

    def load_state_dict(self, state: dict, device=None) -> None:
        count = len(self.params)
        if len(state["m"]) != count or len(state["v"]) != count:
            raise ValueError(f"AdamW.load_state_dict: checkpoint has {len(state['m'])} m and "
                             f"{len(state['v'])} v buffers, expected {count} of each.")
        device_form = {"m": [], "v": []}
        for key in ("m", "v"):
            for i, arr in enumerate(state[key]):
                shape = tuple(self.params[i].data.shape)
                layout = getattr(self.params[i], "_layout", None)
                got = tuple(np.asarray(arr).shape)
                if layout is not None:
                    try:
                        arr = layout.from_stored(arr, v=state["v"][i])
                    except ValueError as exc:
                        raise ValueError(
                            f"AdamW.load_state_dict: {key}[{i}] has shape {got}, which is "
                            f"neither its convolution weight's OIHW shape {layout.oihw} nor a "
                            f"prepared matrix holding it ({exc})") from None
                elif got != shape:
                    raise ValueError(f"AdamW.load_state_dict: {key}[{i}] has shape {got}, which "
                                     f"does not match its parameter's shape {shape}.")
                flat = np.ascontiguousarray(np.asarray(arr, np.float32)).reshape(-1)
                device_form[key].append(torch.from_numpy(flat.copy()).to(self._device))
        t = int(state["t"])
        steps = [int(s) for s in state.get("steps", [t] * count)]
        lr = state.get("lr", self._lr)
        b1, b2 = state.get("betas", (self.b1, self.b2))
        eps = state.get("eps", self.eps)
        weight_decay = state.get("weight_decay", self.weight_decay)
        if len(steps) != count:
            raise ValueError(f"AdamW.load_state_dict: checkpoint has {len(steps)} step counters, "
                             f"expected {count}.")
        if t < 0 or any(s < 0 for s in steps):
            raise ValueError(f"AdamW.load_state_dict: step counts must be >= 0, got t={t}.")
        if not (lr > 0 and eps >= EPS_MIN and weight_decay >= 0 and 0.0 <= b1 < 1.0
                and 0.0 <= b2 < 1.0):
            raise ValueError(f"AdamW.load_state_dict: lr={lr}, betas={(b1, b2)}, eps={eps} or "
                             f"weight_decay={weight_decay} is out of range.")
        self._moments(device_form["m"], device_form["v"], True)
        self._set_steps(t, steps)
        self.lr = lr
        self.b1, self.b2 = float(b1), float(b2)
        self.eps = float(eps)
        self.weight_decay = float(weight_decay)
        self._bias = adam_bias_table(self.b1, self.b2, self._device)
