"""Horovod-style ``DistributedOptimizer`` without the Horovod patch, plus broadcast helpers.

Parity with the patched Horovod 0.18.2 torch integration
(/root/reference/patch_files/horovod/torch/__init__.py:46-250: ``DistributedOptimizer(opt,
grace, named_parameters, backward_passes_per_step)``, ``synchronize``, ``skip_synchronize``,
the double-synchronize warning and the ``zero_grad`` race guard; broadcast_parameters /
broadcast_optimizer_state at 253-403).  The gradient exchange is the bucketed, overlapped
:class:`~grace_amd.parallel.engine.GraceEngine` on RCCL instead of per-parameter Horovod
handles.
"""
from __future__ import annotations

import contextlib
import warnings
from typing import Iterable, Optional, Tuple

import torch
import torch.distributed as dist

from .engine import GraceEngine


class _DistributedOptimizer:
    def __init__(self, optimizer, grace, named_parameters=None, backward_passes_per_step: int = 1,
                 bucket_cap_mb: float = 64.0, overlap: bool = True, sparse_params=(), weights=None,
                 group_collectives=None, watchdog=None, tail_bucket: bool = False):
        self._opt = optimizer
        if named_parameters is None:
            params = [p for g in optimizer.param_groups for p in g["params"]]
            named_parameters = [(f"param.{i}", p) for i, p in enumerate(params)]
        named_parameters = list(named_parameters)
        opt_ids = {id(p) for g in optimizer.param_groups for p in g["params"]}
        missing = [n for n, p in named_parameters if id(p) not in opt_ids]
        if missing:
            raise ValueError(f"named_parameters not in the optimizer: {missing[:5]}")
        self.engine = GraceEngine(named_parameters, grace, bucket_cap_mb=bucket_cap_mb,
                                  backward_passes_per_step=backward_passes_per_step, overlap=overlap,
                                  sparse_params=sparse_params,
                                  grad_sources=weights.grad_sources() if weights is not None else None,
                                  group_collectives=group_collectives, watchdog=watchdog,
                                  tail_bucket=tail_bucket)
        self.weights = weights  # parallel/precision.BF16Weights: refreshed after every step
        # FusedSGD writes the bf16 working copies inside its update kernel (no refresh pass)
        self._fused_refresh = False
        if weights is not None and hasattr(optimizer, "attach_working_copies"):
            optimizer.attach_working_copies(weights)
            self._fused_refresh = True
        self._synchronized = False
        self._should_sync = True

    # attribute passthrough (param_groups, state, ...)
    def __getattr__(self, item):
        return getattr(self._opt, item)

    # an assignment would stay with the wrapper otherwise
    @property
    def max_grad_norm(self):
        return self._opt.max_grad_norm

    @max_grad_norm.setter
    def max_grad_norm(self, bound):
        if not hasattr(self._opt, "max_grad_norm"):
            raise AttributeError(f"{type(self._opt).__name__} does not clip: call clip_grad_norm_ between synchronize and step")
        self._opt.max_grad_norm = bound

    def synchronize(self):
        self.engine.synchronize()
        self._synchronized = True

    @contextlib.contextmanager
    def skip_synchronize(self):
        self._should_sync = False
        try:
            yield
        finally:
            self._should_sync = True

    def step(self, closure=None):
        if self._should_sync:
            if self._synchronized:
                warnings.warn("optimizer.step() called without a new backward after synchronize(); "
                              "use skip_synchronize() to avoid a double exchange")
            else:
                self.synchronize()
        self._synchronized = False
        out = self._opt.step(closure)
        if self.weights is not None and not self._fused_refresh:
            self.weights.refresh()
        return out

    def abort_step(self):
        """Drop a partially launched exchange (e.g. a failed HIP-graph capture) so the next
        eager step starts clean."""
        self.engine.abort_step()
        self._synchronized = False

    def zero_grad(self, set_to_none: bool = True):
        # default (torch's): .grad = None; backward hands every fresh gradient over and ONE native
        # gather launch per bucket copies them in (ResNet-50 Top-K 3534 -> 3645 img/s, BERT QSGD
        # 2221 -> 2307 seq/s vs the memset + per-parameter accumulate of set_to_none=False)
        self.engine.zero_grad(set_to_none)

    def state_dict(self):
        return {"optimizer": self._opt.state_dict(), "grace": self.engine.state_dict()}

    def load_state_dict(self, sd):
        self._opt.load_state_dict(sd["optimizer"])
        self.engine.load_state_dict(sd["grace"])


def DistributedOptimizer(optimizer, grace, named_parameters=None, backward_passes_per_step: int = 1, **kw):
    """Wrap ``optimizer`` so that ``step()`` exchanges gradients through ``grace``."""
    return _DistributedOptimizer(optimizer, grace, named_parameters, backward_passes_per_step, **kw)


def broadcast_parameters(params, root_rank: int = 0, group=None):
    """Bucketed broadcast of a ``state_dict()`` / named parameters (consistent init & resume)."""
    if not (dist.is_available() and dist.is_initialized()) or dist.get_world_size(group) == 1:
        return
    items = list(params.items()) if isinstance(params, dict) else list(params)
    tensors = [t for _, t in items if isinstance(t, torch.Tensor)]
    by = {}
    for t in tensors:
        by.setdefault((t.device, t.dtype), []).append(t)
    for ts in by.values():
        flat = torch.cat([t.detach().reshape(-1) for t in ts])
        dist.broadcast(flat, root_rank, group=group)
        off = 0
        for t in ts:
            n = t.numel()
            with torch.no_grad():
                t.copy_(flat[off:off + n].view_as(t))
            off += n


def _materialize_state(opt) -> None:
    """Create the optimizer's lazily-initialised state with one lr=0 step on zero gradients
    (Horovod's approach, patch_files/horovod/torch/__init__.py:300-330), so every rank holds
    the same state tensors before the broadcast."""
    saved = [g.get("lr") for g in opt.param_groups]
    created = []
    for g in opt.param_groups:
        if "lr" in g:
            g["lr"] = 0.0
        for p in g["params"]:
            if p.requires_grad and p.grad is None:
                p.grad = torch.zeros_like(p)
                created.append(p)
    opt.step()
    for p in created:
        p.grad = None
    for g, lr in zip(opt.param_groups, saved):
        if lr is not None:
            g["lr"] = lr


def broadcast_optimizer_state(optimizer, root_rank: int = 0, group=None):
    """Broadcast every tensor of the optimizer state from ``root_rank``; state that does not
    exist yet is first created on every rank by a no-op step (lr = 0, zero gradients)."""
    if not (dist.is_available() and dist.is_initialized()) or dist.get_world_size(group) == 1:
        return
    opt = getattr(optimizer, "_opt", optimizer)
    if not opt.state_dict()["state"]:
        _materialize_state(opt)
    state = opt.state_dict()["state"]
    tensors = []
    for pid in sorted(state):
        for k in sorted(state[pid]):
            v = state[pid][k]
            if isinstance(v, torch.Tensor):
                tensors.append((f"{pid}.{k}", v))
    broadcast_parameters(tensors, root_rank, group)
