"""Norms around a block, fused with its gate and the scaled residual (``csrc/include/grace_resnorm.h``).

``residual_norm(y, x, weight, bias, gate=g, alpha=a, post=True, ...)`` computes, in one pass over rows
of the last dimension,

    u = post ? N(y; post_weight, post_bias) : y      the norm after the block
    s = a * x + g * u                                the residual stream
    h = N(s; weight, bias)                           the norm before the next block

with N a layer norm or a root-mean-square norm.  Without options it is a plain norm of ``y``; with a
residual alone it is the post-norm step ``N(x + f(x))`` of the encoder.  Everything is computed in fp32
(fp64 for fp64 inputs on the CPU) from the unrounded sum; ``h`` has the type of ``y``, ``s`` that of ``x``.
The backward is one pass too: it keeps an fp32 ``s`` (and ``y`` where a gate or a post norm needs it), or
``x`` and ``y`` where the sum would be rounded to 16 bits; the gradients of weights, biases and shared
gates are summed in a fixed order.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import _native

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check_gate(gate: torch.Tensor, y: torch.Tensor) -> None:
    lead = y.shape[:-1]
    g = gate.shape[:-1] if gate.dim() == y.dim() else (1,) * len(lead) if gate.dim() == 1 else None
    if g is not None and gate.shape[-1] == y.shape[-1]:
        k = 0
        while k < len(lead) and g[k] == lead[k]:
            k += 1
        if all(n == 1 for n in g[k:]):
            return
    raise ValueError(f"residual_norm: a gate of shape {tuple(gate.shape)} for a block of {tuple(y.shape)}: it is "
                     "[width], or the block's shape with 1 in place of trailing dimensions before the last")


def _torch_norm(v, weight, bias, rms, eps):
    if not rms:
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        v = v * weight
    return v if bias is None else v + bias


def residual_norm(y: torch.Tensor, residual: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, *, kind: str = "layer", eps: float = 1e-5,
                  gate: Optional[torch.Tensor] = None, alpha: float = 1.0, post: bool = False,
                  post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                  return_sum: bool = False):
    """``h``, or ``(h, s)`` with ``return_sum`` (the module's docstring has the formulas).

    ``y``: the block's output ``[..., width]``, float32, bfloat16 or float16, width at most 16384 on a GPU.
    ``residual``: the stream, of y's shape, of its type or float32.  ``weight``, ``bias``, ``post_weight``,
    ``post_bias``: ``[width]``; ``gate``: ``[width]``, or y's shape with 1 in place of trailing dimensions
    before the last (``[batch, 1, width]``: one gate a sample); each float32 or of y's type.  ``alpha``
    scales the residual and has no gradient.  Without a residual, a gate and ``post``, ``s`` is ``y``, not a
    copy.  Tensors that are not contiguous are copied first.  Differentiable once."""
    if _native.use_native(y):  # the same refusals, in C++
        out = _native.lib().residual_norm(y, residual, weight, bias, kind, eps, gate, alpha, post, post_weight,
                                          post_bias, return_sum)
        return tuple(out) if return_sum else out[0]
    if kind not in ("layer", "rms"):
        raise ValueError(f"residual_norm: kind {kind!r}: 'layer' or 'rms'")
    if y.dim() < 1 or y.shape[-1] < 1:
        raise ValueError(f"residual_norm: a block of shape {tuple(y.shape)}")
    if not post and (post_weight is not None or post_bias is not None):
        raise ValueError("residual_norm: post_weight and post_bias need post=True")
    if y.dtype not in (*_DTYPES, torch.float64):
        raise TypeError(f"residual_norm: a block of {y.dtype}")
    width = y.shape[-1]
    if residual is None:
        if alpha != 1.0:
            raise ValueError("residual_norm: alpha scales a residual, and there is none")
    else:
        if residual.shape != y.shape or residual.device != y.device:
            raise ValueError(f"residual_norm: a residual of {tuple(residual.shape)} on {residual.device} for a block "
                             f"of {tuple(y.shape)} on {y.device}")
        if residual.dtype not in (y.dtype, torch.float32) or y.dtype == torch.float64 != residual.dtype:
            raise TypeError(f"residual_norm: a residual of {residual.dtype} for a block of {y.dtype}")
    for name, p in (("weight", weight), ("bias", bias), ("post_weight", post_weight), ("post_bias", post_bias),
                    ("gate", gate)):
        if p is None:
            continue
        if p.device != y.device:
            raise ValueError(f"residual_norm: {name} on {p.device}, the block on {y.device}")
        if p.dtype not in (y.dtype, torch.float32):
            raise TypeError(f"residual_norm: {name} of {p.dtype} for a block of {y.dtype}")
        if name != "gate" and p.shape != (width,):
            raise ValueError(f"residual_norm: {name} of shape {tuple(p.shape)} for a width of {width}")
    if gate is not None:
        _check_gate(gate, y)
    rms = kind == "rms"
    wide = torch.float64 if y.dtype == torch.float64 else torch.float32
    w = [None if p is None else p.to(wide) for p in (weight, bias, post_weight, post_bias, gate)]
    s = y.to(wide)
    if post:
        s = _torch_norm(s, w[2], w[3], rms, eps)
    if gate is not None:
        s = s * w[4]
    if residual is not None:
        s = s + alpha * residual.to(wide)
    h = _torch_norm(s, w[0], w[1], rms, eps).to(y.dtype)
    if not return_sum:
        return h
    plain = residual is None and gate is None and not post
    return h, y if plain else s.to(y.dtype if residual is None else residual.dtype)


class ResidualNorm(nn.Module):
    """``forward(y, residual=None, gate=None, return_sum=False)`` is :func:`residual_norm` with this
    module's parameters.  ``weight`` and ``bias`` are named as ``nn.LayerNorm``'s, so state dicts of
    either load into the other; ``post=True`` adds ``post_weight`` (and ``post_bias``)."""

    def __init__(self, width: int, kind: str = "layer", eps: float = 1e-5, bias: bool = True, post: bool = False,
                 alpha: float = 1.0, device=None, dtype=None):
        super().__init__()
        if kind not in ("layer", "rms"):
            raise ValueError(f"ResidualNorm: kind {kind!r}: 'layer' or 'rms'")
        self.width, self.kind, self.eps, self.post, self.alpha = width, kind, eps, post, alpha
        self.weight = nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(width, device=device, dtype=dtype)) if bias else None
        self.post_weight = nn.Parameter(torch.ones(width, device=device, dtype=dtype)) if post else None
        self.post_bias = nn.Parameter(torch.zeros(width, device=device, dtype=dtype)) if post and bias else None

    def forward(self, y, residual=None, gate=None, return_sum: bool = False):
        return residual_norm(y, residual, self.weight, self.bias, kind=self.kind, eps=self.eps, gate=gate,
                             alpha=self.alpha if residual is not None else 1.0, post=self.post,
                             post_weight=self.post_weight, post_bias=self.post_bias, return_sum=return_sum)

    def extra_repr(self) -> str:
        return f"{self.width}, kind={self.kind}, eps={self.eps:g}, post={self.post}, alpha={self.alpha:g}"
