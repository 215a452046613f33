"""``FusedSGD``: torch.optim.SGD with the update done by one native multi-tensor kernel.

Same hyper-parameters, same ``state['momentum_buffer']`` entries (state dicts interchange with
``torch.optim.SGD``), same fp32 arithmetic per element (csrc/kernels/optim.hip).  The kernel
can also write the bf16 working copies of :class:`~grace_amd.parallel.precision.BF16Weights`
in the same pass, replacing ``BF16Weights.refresh()`` -- ``DistributedOptimizer(...,
weights=w)`` arranges that automatically.  CPU tensors (and ``GRACE_AMD_FORCE_TORCH=1``) run
``torch.optim.SGD``'s own functional update.

``max_grad_norm`` clips by the global norm of all gradients of all groups (parallel/clip.py): the
update kernel multiplies every gradient by the factor as it reads it, so the gradients themselves stay
as they are.  The norm of the last step is ``opt.grad_norm``: a 0-dim device tensor, zero in a step
without gradients, None in one without a bound.  The bound is one for all groups; like torch's
hyper-parameters it is an entry of each of them, so copies, pickles and state dicts hold it, and
``opt.max_grad_norm = bound`` changes it.

The learning rate, momentum and bound are read from ``param_groups`` on every ``step()`` call; inside
a captured HIP graph they are frozen at capture time (as for any host scalar), so LR schedules
need eager steps or a re-capture.
"""
from __future__ import annotations

from typing import Dict, Optional

import torch
from torch.optim import SGD

from ..ops import _native


def _dense(t: torch.Tensor) -> bool:
    """Non-overlapping and dense (contiguous up to a permutation of dims, e.g. channels_last)."""
    if t.is_contiguous():
        return True
    expected = 1
    for d in sorted(range(t.dim()), key=lambda d: t.stride(d)):
        if t.size(d) != 1 and t.stride(d) != expected:
            return False
        expected *= t.size(d)
    return True


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Same memory image: equal shapes and equal strides on every dim of size > 1 (a 1x1 conv
    weight in channels_last and its contiguous bucket view differ only on size-1 dims)."""
    return a.shape == b.shape and all(sa == sb for sa, sb, n in zip(a.stride(), b.stride(), a.shape) if n > 1)


def _checked_bound(bound: Optional[float]) -> Optional[float]:
    if bound is not None and not bound >= 0:
        raise ValueError(f"max_grad_norm {bound}: not negative")
    return bound


def _one_bound(groups) -> Optional[float]:
    bounds = {group.get("max_grad_norm") for group in groups}
    if len(bounds) > 1:
        raise ValueError(f"FusedSGD: one max_grad_norm for all groups, not {sorted(bounds, key=str)}")
    return _checked_bound(bounds.pop()) if bounds else None


class FusedSGD(SGD):
    grad_norm: Optional[torch.Tensor] = None

    def __init__(self, params, lr=1e-3, momentum=0.0, dampening=0.0, weight_decay=0.0, nesterov=False, *,
                 maximize: bool = False, max_grad_norm: Optional[float] = None):
        _checked_bound(max_grad_norm)
        super().__init__(params, lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                         nesterov=nesterov, maximize=maximize)
        self._working: Dict[int, torch.Tensor] = {}
        for group in self.param_groups:
            group.setdefault("max_grad_norm", max_grad_norm)
        if _one_bound(self.param_groups) != max_grad_norm:
            raise ValueError("FusedSGD: one max_grad_norm for all groups: give it to the optimizer")
        self.defaults["max_grad_norm"] = max_grad_norm
        # the kernel honours the process-wide communication fault flag (parallel/health.py):
        # allocate it now, before any HIP-graph capture of the step
        devs = {p.device for g in self.param_groups for p in g["params"] if p.is_cuda}
        if devs:
            from . import health

            for d in sorted(devs, key=lambda d: d.index or 0):
                health.init(d)

    @property
    def max_grad_norm(self) -> Optional[float]:
        return _one_bound(self.param_groups)

    @max_grad_norm.setter
    def max_grad_norm(self, bound: Optional[float]) -> None:
        for group in (self.defaults, *self.param_groups):
            group["max_grad_norm"] = _checked_bound(bound)

    def add_param_group(self, param_group) -> None:
        if "max_grad_norm" in self.defaults:  # not while the constructor adds its groups
            _one_bound([self.defaults, {**self.defaults, **param_group}])
        super().add_param_group(param_group)

    def __setstate__(self, state) -> None:
        """After load_state_dict (groups without a bound, as torch.optim.SGD's, keep this optimizer's), copies and
        pickles (whose working copies have to be attached again)."""
        own = self.__dict__.get("defaults") or state.get("defaults", {})
        for group in state["param_groups"]:
            group.setdefault("max_grad_norm", own.get("max_grad_norm"))
        bound = _one_bound(state["param_groups"])
        super().__setstate__(state)
        self.defaults["max_grad_norm"] = bound
        self.__dict__.setdefault("_working", {})

    def attach_working_copies(self, weights) -> None:
        """Write ``weights``' bf16 working copies in the update kernel (BF16Weights)."""
        self._working = {id(master): work for _, _, master, work in weights.entries}

    @property
    def writes_working_copies(self) -> bool:
        return bool(self._working)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        bound = self.max_grad_norm
        self.grad_norm = None
        factor = self._clip_factor(float(bound)) if bound is not None else None
        for group in self.param_groups:
            native, rest = [], []
            on = {}  # device -> whether its native path runs
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise RuntimeError("FusedSGD does not support sparse gradients")
                dev = p.device
                if dev not in on:
                    on[dev] = _native.native_on(dev)
                ok = (on[dev] and p.dtype == torch.float32 and g.dtype == torch.float32
                      and (p.is_contiguous() and g.is_contiguous() and p.shape == g.shape
                           or _same_layout(g, p) and _dense(p)))
                (native if ok else rest).append(p)
            if native:
                self._native_step(group, native, factor)
            if rest:
                self._torch_step(group, rest, factor)
        return loss

    def _clip_factor(self, bound: float) -> Optional[torch.Tensor]:
        from .clip import _check, _norm_and_factor, _unique

        params = [p for g in self.param_groups for p in g["params"]]
        if params and _native.use_native(params[0]):
            out = _native.lib().grad_clip(params, 2, bound, False)
            if out is not None:
                self.grad_norm = out[0]
                return out[1]
        grads = _unique([p.grad for p in params if p.grad is not None])
        if not grads:
            self.grad_norm = torch.zeros((), device=params[0].device if params else None)
            return None
        _check(grads)
        self.grad_norm, factor = _norm_and_factor(grads, 2, bound)
        return factor

    def _native_step(self, group, params, factor):
        mom = group["momentum"]
        first, later = [], []
        for p in params:
            st = self.state[p]
            if mom != 0 and st.get("momentum_buffer") is None:
                st["momentum_buffer"] = torch.empty_like(p)  # same strides as p
                first.append(p)
            else:
                later.append(p)
        # one launch per device (the kernel reads that device's communication fault word)
        devs = {}
        for ps, is_first in ((first, True), (later, False)):
            for p in ps:
                devs.setdefault((p.device, is_first), []).append(p)
        for (dev, is_first), ps in devs.items():
            bufs = [self.state[p].get("momentum_buffer") if mom != 0 else None for p in ps]
            w16 = [self._working_for(p) for p in ps] if self._working else [None] * len(ps)
            _native.lib().sgd_step(ps, [p.grad for p in ps], bufs, w16, float(group["lr"]), float(mom),
                                   float(group["dampening"]), float(group["weight_decay"]),
                                   bool(group["nesterov"]), bool(group.get("maximize", False)), is_first,
                                   None if factor is None else factor.to(dev, torch.float32))
            for p, w in zip(ps, w16):  # working copies the kernel could not write (other strides)
                if w is None and id(p) in self._working:
                    self._working[id(p)].copy_(p)

    def _working_for(self, p) -> Optional[torch.Tensor]:
        if not self._working:
            return None
        w = self._working.get(id(p))
        return w if (w is not None and _same_layout(w, p)) else None

    def _torch_step(self, group, params, factor):
        from torch.optim.sgd import sgd as functional_sgd

        bufs = [self.state[p].get("momentum_buffer") for p in params]
        grads = [p.grad for p in params]
        if factor is not None:
            # widened by hand: a product of a 16-bit tensor and a device scalar is taken with the scalar in 16 bits
            grads = [(g.to(factor.dtype) * factor.to(g.device)).to(g.dtype) for g in grads]
        functional_sgd(params, grads, bufs, weight_decay=group["weight_decay"],
                       momentum=group["momentum"], lr=group["lr"], dampening=group["dampening"],
                       nesterov=group["nesterov"], maximize=group.get("maximize", False), foreach=False)
        if group["momentum"] != 0:
            for p, b in zip(params, bufs):
                self.state[p]["momentum_buffer"] = b
        for p in params:
            w = self._working.get(id(p))
            if w is not None:
                w.copy_(p)
