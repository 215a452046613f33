"""The global gradient norm over many tensors, and clipping by it (``csrc/kernels/gradnorm.hip``).

``clip_grad_norm_`` has the formula of ``torch.nn.utils.clip_grad_norm_`` and its arguments but for
``foreach``, with 1, 2 and inf for ``norm_type``: gradients are multiplied by ``min(1, max_norm / (norm + 1e-6))``.  The norm is summed in fp64 over all
tensors, whatever their types, in one launch per 240 tensors and in a fixed order; nothing waits for
the host, so the call can be captured into a HIP graph.  A factor of one leaves the gradients' memory
untouched.

In data-parallel training the norm is that of the exchanged gradients, the same on every rank:

    opt.synchronize()                                  # DistributedOptimizer
    clip_grad_norm_(model.parameters(), 1.0)
    with opt.skip_synchronize():
        opt.step()

(With :class:`~grace_amd.parallel.precision.BF16Weights` the exchanged gradients are those of
``weights.master_parameters(model)``; the model's own parameters hold the local ones.)

``FusedSGD(..., max_grad_norm=1.0)`` does the same inside its update, without writing the clipped
gradients.
"""
from __future__ import annotations

import math
from typing import Iterable, List, Tuple, Union

import torch

from ..ops import _native
from .fused_sgd import _dense

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_KINDS = {math.inf: 0, 1.0: 1, 2.0: 2}


def _kind(norm_type) -> int:
    try:
        return _KINDS[float(norm_type)]
    except KeyError:
        raise ValueError(f"norm_type {norm_type}: 1, 2 or inf") from None


def _check(grads: List[torch.Tensor]) -> None:
    for g in grads:
        if g.layout != torch.strided:
            raise TypeError(f"gradient norm: a {g.layout} gradient: strided ones only")
        if not g.is_floating_point():
            raise TypeError(f"gradient norm: a gradient of {g.dtype}")


def _native_ok(g: torch.Tensor) -> bool:
    return g.dtype in _DTYPES and _native.use_native(g)


def _memory(g: torch.Tensor):
    """Equal for two tensors that show the same elements, in whatever order."""
    if g.layout != torch.strided or g.numel() == 0:
        return id(g)
    places = (g.numel(),) if _dense(g) else tuple(sorted((s, n) for s, n in zip(g.stride(), g.shape) if n > 1))
    return g.device, g.data_ptr(), g.dtype, places


def _apart(grads: List[torch.Tensor]) -> bool:
    """No two of these tensors, some with gaps between their elements, share any of their memory."""
    unit = min(g.element_size() for g in grads)
    base = min(g.data_ptr() for g in grads)
    shown = torch.zeros((max(_end(g) for g in grads) - base) // unit, dtype=torch.int16)
    for g in grads:
        k = g.element_size() // unit
        shown.as_strided((*g.shape, k), (*(s * k for s in g.stride()), 1), (g.data_ptr() - base) // unit).add_(1)
    return int(shown.max()) <= 1


def _end(g: torch.Tensor) -> int:
    return g.data_ptr() + (1 + sum(s * (n - 1) for s, n in zip(g.stride(), g.shape))) * g.element_size()


def _expanded(g: torch.Tensor) -> bool:
    return any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape))


def _unique(grads: List[torch.Tensor]) -> List[torch.Tensor]:
    """Every piece of memory once: one that several tensors show counts once and is scaled once, as in the kernels'
    own list.  Tensors that share a part of their memory are refused."""
    once = list({_memory(g): g for g in grads}.values())
    by = {}
    for g in once:
        if g.layout == torch.strided and g.numel() > 0 and not _expanded(g):
            by.setdefault(g.device, []).append(g)
    for on in by.values():
        runs, end = [], 0  # tensors whose spans of memory meet
        for g in sorted(on, key=lambda g: g.data_ptr()):
            if g.data_ptr() < end:
                runs[-1].append(g)
            else:
                runs.append([g])
            end = max(end, _end(g))
        for run in runs:
            if len(run) > 1 and (all(_dense(g) for g in run) or not _apart(run)):
                raise RuntimeError("gradient norm: two tensors overlap")
    return once


def _groups(grads: List[torch.Tensor]):
    """{device: (tensors for the kernels, other tensors)}"""
    by = {}
    for g in grads:
        by.setdefault(g.device, ([], []))[0 if _native_ok(g) else 1].append(g)
    return by


def _packed(g: torch.Tensor) -> torch.Tensor:
    """g, or a contiguous copy where its elements lie apart or overlap."""
    return g if _dense(g) else g.contiguous()


def _torch_part(g: torch.Tensor, kind: int) -> torch.Tensor:
    if g.numel() == 0:
        return torch.zeros((), dtype=torch.float64, device=g.device)
    a = g.detach().double()
    return a.abs().max() if kind == 0 else a.abs().sum() if kind == 1 else a.square().sum()


def _parts(grads: List[torch.Tensor], kind: int) -> List[torch.Tensor]:
    """1-D fp64 tensors of partial values, one or two for each device."""
    parts = []
    for native, other in _groups(grads).values():
        if native:
            parts.append(_native.lib().grad_norm_parts([_packed(g) for g in native], kind))
        if other:
            parts.append(torch.stack([_torch_part(g, kind) for g in other]))
    return parts


def _norm_and_factor(grads: List[torch.Tensor], kind: int, max_norm: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """0-dim norm and factor on the first gradient's device."""
    dev = grads[0].device
    parts = [p if p.device == dev else p.to(dev) for p in _parts(grads, kind)]
    part = parts[0] if len(parts) == 1 else torch.cat(parts)
    if _native.native_on(dev) and not any(g.dtype == torch.float64 for g in grads):
        out = _native.lib().grad_norm_finish(part, kind, max_norm)
        return out[0], out[1]
    norm = part.max() if kind == 0 else part.sum() if kind == 1 else part.sum().sqrt()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    dtype = torch.float64 if any(g.dtype == torch.float64 for g in grads) else torch.float32
    return norm.to(dtype), factor.to(dtype)


def _scale(grads: List[torch.Tensor], factor: torch.Tensor) -> None:
    for dev, (native, other) in _groups(grads).items():
        f = factor if factor.device == dev else factor.to(dev)
        if native:
            dense = [_packed(g) for g in native]
            _native.lib().grad_scale(dense, f.float())
            for g, d in zip(native, dense):
                if d is not g:
                    g.copy_(d)
        for g in other:
            g.copy_(g.to(f.dtype) * f) if g.dtype in (torch.bfloat16, torch.float16) else g.mul_(f)


def _grads_of(parameters) -> List[torch.Tensor]:
    grads = _unique([p.grad for p in parameters if p.grad is not None])
    _check(grads)
    if any(_expanded(g) for g in grads):
        raise ValueError("clip_grad_norm_: an expanded gradient: several of its elements share memory")
    return grads


@torch.no_grad()
def grad_norm(tensors: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all tensors taken as one vector: a 0-dim tensor (fp32; fp64 if any tensor is) on the
    first tensor's device.  ``norm_type``: 1, 2 or inf.  Memory that is given twice, by the same tensor or by
    two views of all its elements, counts once; tensors that share a part of theirs are refused."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    kind, tensors = _kind(norm_type), _unique(tensors)
    _check(tensors)
    if not tensors:
        return torch.tensor(0.0)
    return _norm_and_factor(tensors, kind, 1.0)[0]


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the parameters' ``.grad`` in place by ``min(1, max_norm / (norm + 1e-6))`` and return the norm
    before it (0-dim).  ``norm_type``: 1, 2 or inf.  A shared parameter or gradient counts once, also as two
    views; gradients that share a part of their memory are refused.  A non-finite norm makes the gradients NaN or
    zero, as torch's function does; ``error_if_nonfinite`` raises instead, before anything is scaled, for
    which it waits for the device."""
    kind, max_norm = _kind(norm_type), float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm {max_norm}: not negative")
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if not error_if_nonfinite and parameters and _native.use_native(parameters[0]):
        out = _native.lib().grad_clip(parameters, kind, max_norm, True)
        if out is not None:
            return out[0]
    grads = _grads_of(parameters)
    if not grads:
        return torch.tensor(0.0)
    norm, factor = _norm_and_factor(grads, kind, max_norm)
    if error_if_nonfinite and not bool(torch.isfinite(norm)):
        raise RuntimeError(f"The total norm of order {float(norm_type)} for gradients is non-finite, so it cannot be "
                           "clipped")
    _scale(grads, factor)
    return norm
