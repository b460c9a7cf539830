"""AdamW over many tensors in one launch, moments in 32 bits or in 8 (no reference
counterpart: the reference leaves the training step to the caller).

    adamw_step(params, grads, exp_avgs, exp_avg_sqs, step=t, lr=...)   the step
    AdamW(params, lr=..., bits=8).step()                               its state kept

An 8-bit moment is a pair (codes, scales): codes float8_e4m3fn in the parameter's
shape, scales float32 (ceil(n / 256),), value = code * scale over runs of 256
values; the second moment's codes are those of its square root.
"""
from __future__ import annotations

import struct
from itertools import repeat

import torch

from . import _lib
from .encoder import _run
from .errors import ArgumentError, DimensionMismatch

BLOCK = 256
_FLOAT = {torch.float32, torch.float16, torch.bfloat16}
_HALF = {torch.float16, torch.bfloat16}
# one fms_adamw_tensor: p, g, copy, m, v, m_scales, v_scales, n, and the codes of three types
_pack = struct.Struct("=7QqiiiI").pack


_get_device = torch.Tensor.get_device
_is_contiguous = torch.Tensor.is_contiguous
_numel = torch.Tensor.numel
_data_ptr = torch.Tensor.data_ptr


def _checked(dev, ts):
    # a model has hundreds of tensors, and this runs every step: whole-list calls
    if set(map(_get_device, ts)) - {dev.index}:
        raise ArgumentError("adamw_step: all tensors must live on one CUDA device")
    if not all(map(_is_contiguous, ts)):
        raise ArgumentError("adamw_step: tensors are updated in place and must be contiguous")
    return list(map(_data_ptr, ts))


def _dtypes(ts):
    return [t.dtype for t in ts]


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr=1e-3, betas=(0.9, 0.999),
               eps=1e-8, weight_decay=1e-2, seed=0, copies=None, grad_scale=None):
    """One AdamW step (decoupled weight decay) in place over lists of tensors:

        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
        p = (1 - lr wd) p - lr / (1 - b1^step) * m / (sqrt(v) / sqrt(1 - b2^step) + eps)

    params and grads are float32, float16 or bfloat16.  exp_avgs and exp_avg_sqs
    are lists of float32 tensors, or of (codes, scales) pairs of 8-bit moments
    (`moments8`), whose codes are rounded stochastically by (seed, step).  copies
    (16-bit tensors, or None) receive the new parameters in their type.  step
    counts from 1.  grad_scale, a float32 tensor of one value, multiplies the
    gradients (a clipping factor, an inverse loss scale)."""
    _take(_plan(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay, seed, copies, grad_scale))


def _plan(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas, eps, weight_decay, seed, copies, grad_scale):
    """Checks one step's arguments: its device, the tensors that it writes, the call's arguments."""
    params, grads = list(params), list(grads)
    exp_avgs, exp_avg_sqs = list(exp_avgs), list(exp_avg_sqs)
    n = len(params)
    copies = None if copies is None else list(copies)
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n) or \
            (copies is not None and len(copies) != n):
        raise DimensionMismatch("adamw_step: lists must have one entry per parameter")
    b1, b2 = betas
    if not (0 <= b1 < 1 and 0 <= b2 < 1) or not eps >= 0 or int(step) < 1:
        raise ArgumentError("adamw_step: betas must be in [0, 1), eps >= 0 and step >= 1")
    if n == 0:
        return None
    dev = params[0].device
    if dev.type != "cuda":
        raise ArgumentError("adamw_step runs on CUDA tensors only")
    eight = isinstance(exp_avgs[0], (tuple, list))
    states, scales = exp_avgs + exp_avg_sqs, []
    if eight:
        if not all(isinstance(s, (tuple, list)) and len(s) == 2 for s in states):
            raise ArgumentError("adamw_step: moments must all be tensors or all (codes, scales)")
        scales, states = [s[1] for s in states], [s[0] for s in states]
        if set(_dtypes(scales)) != {torch.float32}:
            raise ArgumentError("adamw_step: scales of 8-bit moments must be float32")
    elif not all(isinstance(s, torch.Tensor) for s in states):
        raise ArgumentError("adamw_step: moments must all be tensors or all (codes, scales)")
    want = torch.float8_e4m3fn if eight else torch.float32
    if set(_dtypes(states)) != {want}:
        raise ArgumentError(f"adamw_step: moments must hold {want}")
    pt, gt = _dtypes(params), _dtypes(grads)
    if not set(pt + gt) <= _FLOAT:
        raise ArgumentError("adamw_step: parameters and gradients must be float32, float16 or bfloat16")
    ct = None if copies is None else _dtypes(copies)
    if copies is not None and not set(ct) <= _HALF:
        raise ArgumentError("adamw_step: copies must be float16 or bfloat16")
    sizes = list(map(_numel, params))
    if list(map(_numel, grads)) != sizes or list(map(_numel, states)) != sizes + sizes or \
            (copies is not None and list(map(_numel, copies)) != sizes):
        raise DimensionMismatch("adamw_step: gradients, moments and copies must have their parameter's size")
    at = _checked(dev, params + grads + states + (copies or []))
    p, g, m, v, c = at[:n], at[n:2 * n], at[2 * n:3 * n], at[3 * n:4 * n], at[4 * n:]
    ms = vs = none = repeat(0)
    if eight:
        blocks = [-(-s // BLOCK) for s in sizes]
        if list(map(_numel, scales)) != blocks + blocks:
            raise DimensionMismatch("adamw_step: 8-bit moments need one scale per 256 values")
        at = _checked(dev, scales)
        ms, vs = at[:n], at[n:]
    code = _lib.DTYPE_CODE.__getitem__
    table = b"".join(map(_pack, p, g, c or none, m, v, ms, vs, sizes, map(code, pt), map(code, gt),
                         none if ct is None else map(code, ct), none))
    if grad_scale is not None:
        if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1:
            raise ArgumentError("adamw_step: grad_scale must be a float32 tensor of one value")
        _checked(dev, [grad_scale])
    # Two entries that write the same memory would race in the kernel.  (Empty tensors have
    # no address, and a copy may be its parameter.)
    lists = [p, m, v, c] + ([ms, vs] if eight else [])
    starts = sum(lists, [])
    if len(set(starts)) < len(starts):
        lists[3] = [0 if a == b else a for a, b in zip(c, p)]
        starts = [a for ts in lists for a, s in zip(ts, sizes) if s and a]
        if len(set(starts)) < len(starts):
            raise ArgumentError("adamw_step: a tensor that is written is named twice")
    written = params + states + scales + (copies or [])
    return dev, written, (8 if eight else 32, n, table, int(step), float(lr), float(b1), float(b2),
                          float(eps), float(weight_decay), int(seed) & 0xFFFFFFFF,
                          None if grad_scale is None else grad_scale.data_ptr())


def _take(plan):
    if plan is not None:
        dev, written, args = plan
        torch.autograd.graph.increment_version(written)
        _run("fms_adamw_step", dev, *args)


def moments8(p):
    """A zero 8-bit moment (codes, scales) of parameter p."""
    return (torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device),
            torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device))


def _parts(moment):
    return list(moment) if isinstance(moment, (tuple, list)) else [moment]


def _copy(moment, device=None):
    if moment is None:
        return None
    c = [t.detach().to(t.device if device is None else device, copy=True).contiguous() for t in _parts(moment)]
    return tuple(c) if isinstance(moment, (tuple, list)) else c[0]


class AdamW:
    """AdamW over a list of parameters, its moments kept in `bits` (32 or 8) each.

    `step()` reads each parameter's .grad (or the list given); parameters without
    one are left alone.  With `copies`, 16-bit tensors beside float32 parameters
    receive the new values (the weights that the model computes with).  Moments
    are made at a parameter's first step."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32,
                 seed=0, copies=None):
        if bits not in (32, 8):
            raise ArgumentError(f"AdamW: bits must be 32 or 8, got {bits!r}")
        self.params = list(params)
        self.copies = None if copies is None else list(copies)
        if self.copies is not None and len(self.copies) != len(self.params):
            raise DimensionMismatch("AdamW: one copy per parameter")
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.bits, self.seed = bits, seed
        self.steps = [0] * len(self.params)  # each parameter's own: its bias correction
        self.exp_avgs = [None] * len(self.params)
        self.exp_avg_sqs = [None] * len(self.params)

    def _moment(self, p):
        return moments8(p) if self.bits == 8 else \
            torch.zeros(p.shape, dtype=torch.float32, device=p.device)

    def step(self, grads=None, grad_scale=None):
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            raise DimensionMismatch("AdamW: one gradient per parameter")
        groups = {}  # by the step that they are at
        for k, g in enumerate(grads):
            if g is not None:
                groups.setdefault(self.steps[k] + 1, []).append(k)
        plans = []  # all of them are checked before any is taken: a refused step changes nothing
        for t, ks in sorted(groups.items()):
            pick = lambda ts: [ts[k] for k in ks]  # noqa: B023, E731
            m, v = ([s[k] if s[k] is not None else self._moment(self.params[k]) for k in ks]
                    for s in (self.exp_avgs, self.exp_avg_sqs))
            plans.append((t, ks, m, v, _plan(
                pick(self.params), pick(grads), m, v, t, self.lr, self.betas, self.eps,
                self.weight_decay, self.seed, None if self.copies is None else pick(self.copies), grad_scale)))
        for t, ks, m, v, plan in plans:
            _take(plan)
            for k, a, b in zip(ks, m, v):
                self.exp_avgs[k], self.exp_avg_sqs[k], self.steps[k] = a, b, t

    def zero_grad(self):
        for p in self.params:
            p.grad = None

    def state_dict(self):
        """A copy of the state: later steps do not change it."""
        return {"steps": list(self.steps), "bits": self.bits, "exp_avgs": list(map(_copy, self.exp_avgs)),
                "exp_avg_sqs": list(map(_copy, self.exp_avg_sqs))}

    def load_state_dict(self, state):
        """Takes up a copy of a state of this width and these parameters' sizes, from any
        device; one that does not fit is refused and changes nothing."""
        n = len(self.params)
        steps, moments = list(state["steps"]), [list(state["exp_avgs"]), list(state["exp_avg_sqs"])]
        if state["bits"] != self.bits or any(len(s) != n for s in (steps, *moments)):
            raise ArgumentError("AdamW: the state is of another width or number of parameters")
        want = [torch.float8_e4m3fn, torch.float32] if self.bits == 8 else [torch.float32]
        for p, t, m, v in zip(self.params, steps, *moments):
            if t < 0 or (m is None) != (v is None) or (m is None) != (t == 0):
                raise ArgumentError("AdamW: the state's counts and moments do not belong together")
            sizes = [p.numel(), -(-p.numel() // BLOCK)][:len(want)]
            for s in (m, v) if m is not None else ():
                parts = _parts(s)
                if len(parts) != len(want) or _dtypes(parts) != want:
                    raise ArgumentError(f"AdamW: moments of {self.bits} bits must hold {want}")
                if list(map(_numel, parts)) != sizes:
                    raise DimensionMismatch("AdamW: a moment is not of its parameter's size")
        self.exp_avgs, self.exp_avg_sqs = ([_copy(s, p.device) for s, p in zip(m, self.params)] for m in moments)
        self.steps = steps
