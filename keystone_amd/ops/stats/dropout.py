"""Dropout of features during training, from a counter.

Whether element i of a batch is kept is a function of ``(seed, step, i)``, so
the CPU and the GPU keep the same ones and no mask is stored: the gradient
with respect to the input is the same call on the output's gradient.  The
generator is Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): key = seed,
counter = (i div 8, step), 16 bits an element.
"""

from __future__ import annotations

import torch

from ...utils.derivatives import differentiated

__all__ = ["dropout"]

_LOW = 0xFFFFFFFF


def _signed(x: int) -> int:
    return x - (1 << 64) if x >= 1 << 63 else x


def _words(blocks: torch.Tensor, seed: int, step: int):
    c = [blocks & _LOW, (blocks >> 32) & _LOW,
         torch.full_like(blocks, step & _LOW),
         torch.full_like(blocks, step >> 32)]
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(10):
        # 64-bit products wrap, so that their upper halves come out signed
        a = c[0] * _signed(0xD2511F53)
        b = c[2] * _signed(0xCD9E8D57)
        c = [((b >> 32) & _LOW) ^ c[1] ^ k0, b & _LOW,
             ((a >> 32) & _LOW) ^ c[3] ^ k1, a & _LOW]
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return c


def dropout(x: torch.Tensor, p: float, seed: int, step: int = 0
            ) -> torch.Tensor:
    """Zeros each element with chance ``p`` (to a multiple of 2^-16) and
    scales the others so that the mean stays."""
    from ... import hip
    # the kernel keeps nothing for autograd
    if x.is_cuda and x.dtype in (torch.float32, torch.bfloat16, torch.float16) \
            and not differentiated(x) and hip.gpu_ready():
        return hip.dropout(x, p, seed, step)
    if not (0 <= seed < 2 ** 64 and 0 <= step < 2 ** 64):
        raise ValueError("dropout: expected a seed and a step in [0, 2^64), "
                         f"got {seed} and {step}")
    n, t = x.numel(), hip.dropout_threshold(p)
    words = _words(torch.arange(-(-n // 8), device=x.device), seed, step)
    bits = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 1)
    keep = bits.reshape(-1)[:n].reshape(x.shape) >= t
    wide = x.to(torch.promote_types(x.dtype, torch.float32))
    scale = torch.tensor(65536 / (65536 - t), dtype=wide.dtype)
    return torch.where(keep, wide * scale.to(x.device),
                       torch.zeros((), dtype=wide.dtype, device=x.device)
                       ).to(x.dtype)
