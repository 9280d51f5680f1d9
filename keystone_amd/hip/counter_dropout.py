"""Dropout on the GPU from a counter-based generator (dropout.hip)."""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _launch, _load, _ptr

__all__ = ["dropout", "dropout_threshold"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def dropout_threshold(p: float) -> int:
    """Of 65536 equally likely numbers those below this one drop."""
    t = round(p * 65536) if 0.0 <= p < 1.0 else -1
    if not 0 <= t < 65536:
        raise ValueError(f"dropout: expected a chance p in [0, 1 - 2^-17), "
                         f"got {p}")
    return t


def dropout(x: torch.Tensor, p: float, seed: int,
            step: Union[int, torch.Tensor] = 0,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Zeros each element with chance ``p`` and scales the others so that the
    mean stays.  Which ones is a function of ``(seed, step)`` and the
    element's place in ``x`` alone: the gradient is ``dropout(dy, p, seed,
    step)``, and no mask is kept, nor anything for autograd.  What is dropped is
    zero whatever it held.

    ``step``: a number below 2^64, or an int64 tensor of one element on x's
    device, which a captured graph reads at each replay.  ``out`` may be
    ``x``."""
    _load()
    if not x.is_cuda:
        raise RuntimeError("dropout.x: expected CUDA tensor")
    if x.dtype not in _TYPES:
        raise RuntimeError(f"dropout.x: expected float32, bfloat16 or "
                           f"float16, got {x.dtype}")
    t = dropout_threshold(p)
    if not 0 <= seed < 2 ** 64:
        raise ValueError(f"dropout: expected a seed in [0, 2^64), got {seed}")
    at = None
    if isinstance(step, torch.Tensor):
        if step.device != x.device or step.dtype != torch.int64 \
                or step.numel() != 1:
            raise RuntimeError("dropout.step: expected one int64 element on "
                               f"{x.device}, got {tuple(step.shape)} "
                               f"{step.dtype} on {step.device}")
        at, step = step, 0
    elif not 0 <= step < 2 ** 64:
        raise ValueError(f"dropout: expected a step in [0, 2^64), got {step}")
    if x.is_neg():                # a sign that torch has put off
        x = x.resolve_neg()
    if out is None:
        x = x.contiguous()
        out = torch.empty_like(x)
    else:
        if out.shape != x.shape or out.dtype != x.dtype \
                or out.device != x.device or not out.is_contiguous() \
                or out.is_neg():
            raise RuntimeError("dropout.out: expected a contiguous tensor of "
                               "x's shape, type and device, no negated view")
        x = x.contiguous()
        lo, size = out.data_ptr(), x.numel() * x.element_size()
        if 0 < abs(x.data_ptr() - lo) < size:
            raise ValueError("dropout: out overlaps x")
    _launch("ks_dropout", x.device, x.data_ptr(), out.data_ptr(), x.numel(),
            _TYPES[x.dtype], t, 65536 / (65536 - t), seed, step, _ptr(at))
    return out
