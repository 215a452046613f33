"""Embedding lookup with scaling, and its gradient by sorted tokens (``csrc/kernels/embed.hip``).

``embedding(ids, weight, scale)`` is ``round(scale * weight[ids])``; its gradient sums the rows of the
output's gradient over equal tokens in fp32 (fp64 for an fp64 table on the CPU), in token order, and
rounds once to the table's type.  On a GPU the tokens are sorted by row and runs of equal tokens are
summed in a fixed order: no atomics, the same result on every call.  Every row of the gradient is written,
untouched rows as zeros.

A token outside the table raises ``IndexError`` on the CPU.  On a GPU, where that check would
need a device synchronisation, its output row is NaN and it adds nothing to the gradient.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _native


def _plain(ids, weight, scale, padding_idx, dtype):
    """With rows of NaN, and no gradient, for tokens outside the table."""
    wide = weight if weight.dtype == torch.float64 else weight.float()
    inside = (ids >= 0) & (ids < weight.shape[0])
    y = F.embedding(torch.where(inside, ids, 0), wide, padding_idx) * float(scale)
    return torch.where(inside[..., None], y, float("nan")).to(dtype)


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None,
              dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``round(scale * weight[ids])`` of shape ``[*ids.shape, width]``.

    ``ids``: int64 or int32, any shape and strides.  ``weight``: ``[rows, width]``, float32, bfloat16 or
    float16 (on the CPU float64 too), on a GPU at most 2^21 wide.  ``dtype``: the output's type (default: the table's).
    ``padding_idx`` (negative: from the end) names a row that gets no gradient.  Differentiable once, in
    ``weight``."""
    if _native.use_native(weight):
        return _native.lib().embedding(ids, weight, scale, padding_idx, dtype)  # the same refusals, in C++
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"embedding: ids must be int64 or int32, got {ids.dtype}")
    if weight.dim() != 2:
        raise ValueError(f"embedding: the table must be [rows, width], got {tuple(weight.shape)}")
    if ids.device != weight.device:
        raise ValueError(f"embedding: ids on {ids.device}, table on {weight.device}")
    rows = weight.shape[0]
    if rows == 0 and ids.numel() > 0:
        raise ValueError("embedding: the table has no rows")
    if padding_idx is not None and not -rows <= padding_idx < rows:
        raise ValueError(f"embedding: padding_idx {padding_idx} outside a table of {rows} rows")
    out = weight.dtype if dtype is None else dtype
    for t in (weight.dtype, out):
        if t not in (torch.float32, torch.bfloat16, torch.float16, torch.float64):
            raise TypeError(f"embedding: float32, bfloat16 or float16, got {weight.dtype} -> {out}")
    if weight.is_cuda and rows > 0:  # without the kernels: what they give, and torch reads nothing behind the table
        return _plain(ids, weight, scale, padding_idx, out)
    wide = weight if weight.dtype == torch.float64 else weight.float()
    return (F.embedding(ids, wide, padding_idx) * float(scale)).to(out)


class ScaledEmbedding(nn.Embedding):
    """Drop-in ``nn.Embedding`` (same parameter, same state dict) on the native kernels, with a factor
    on the looked-up rows.  ``max_norm``, ``scale_grad_by_freq`` and ``sparse`` are refused."""

    def __init__(self, *args, scale: float = 1.0, **kw):
        super().__init__(*args, **kw)
        if self.max_norm is not None or self.scale_grad_by_freq or self.sparse:
            raise ValueError("ScaledEmbedding: max_norm, scale_grad_by_freq and sparse are not supported")
        self.scale = float(scale)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return embedding(ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return super().extra_repr() + f", scale={self.scale:g}"
