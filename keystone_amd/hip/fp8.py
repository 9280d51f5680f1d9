"""Linear maps with 8-bit operands (fp8_linear.hip).

A block of 128 neighbours along the inner dimension (of a row of ``X``, of a
column of ``W``) is held as e4m3 numbers times a power of two, the least that
brings the block's largest under 448.  Scaling by a power of two is exact, so
an element is off by at most 2^-4 of itself (or 2^-10 of its block's scale,
where that is more), and the matrix instruction applies the scales itself.
Scales are at least 2^-117.  A block that holds an infinity or a NaN is NaN
throughout.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _launch, _load, _ptr

__all__ = ["Fp8Weight", "fp8_pack", "fp8_linear", "fp8_round"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX = 2 ** 31 - 2048      # rows
_MAX_INNER = 2 ** 26


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """Whole and from 16 bytes on, as the kernels read it."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class Fp8Weight:
    """``W`` [K, N] in 8 bits, laid out as the matrix instruction reads it:
    ``data`` [N/16, K/128, 2048] bytes and ``scales`` [N/16, K/512, 64]
    bytes, 127 + exponent (127 past the end), with sides rounded up."""

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, K: int,
                 N: int):
        tiles, kb = -(-N // 16), -(-K // 128)
        for t, shape in ((data, (tiles, kb, 2048)),
                         (scales, (tiles, -(-kb // 4), 64))):
            if t.shape != shape or t.dtype != torch.uint8:
                raise ValueError(f"Fp8Weight: expected uint8 {shape} for W "
                                 f"[{K}, {N}], got {t.dtype} "
                                 f"{tuple(t.shape)}")
        self.data, self.scales = _aligned(data), _aligned(scales)
        self.K, self.N = K, N

    def to(self, device) -> "Fp8Weight":
        return Fp8Weight(self.data.to(device), self.scales.to(device), self.K,
                         self.N)

    def dequantise(self) -> torch.Tensor:
        """The [K, N] float32 matrix that the bytes stand for."""
        tiles, kb = self.data.shape[:2]
        # lane 16 g + r of plane p holds row r's k = 32 (2 p + h) + 8 g + i
        q = self.data.view(tiles, kb, 2, 4, 16, 2, 8) \
            .permute(0, 4, 1, 2, 5, 3, 6).reshape(tiles * 16, kb, 128)
        e = self.scales.view(tiles, -(-kb // 4), 16, 4).permute(0, 2, 1, 3) \
            .reshape(tiles * 16, -(-kb // 4) * 4)[:, :kb].to(torch.int32) - 127
        q = q.contiguous().view(torch.float8_e4m3fn).to(torch.float32)
        q = q * _power_of_two(e).unsqueeze(2)
        return q.flatten(1)[:self.N, :self.K].t()


def _power_of_two(e: torch.Tensor) -> torch.Tensor:
    """float32 2^e of int32 e in [-126, 127], exactly (torch.ldexp goes by
    way of pow, which need not be)."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(x: torch.Tensor):
    """e4m3 values [rows, K/128, 128] and exponents [rows, K/128] of a
    float32 matrix, in torch."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 128))
    x = x.reshape(x.shape[0], x.shape[1] // 128, 128)
    top = x.abs().amax(2)
    bad = ~top.isfinite()
    m, e = torch.frexp(torch.where(bad, torch.zeros_like(top), top))
    e = torch.where(m > 0, (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-117),
                    torch.zeros_like(e))
    q = x * _power_of_two(-e).unsqueeze(2)
    q = torch.where(bad.unsqueeze(2), torch.full_like(q, float("nan")), q)
    return q.to(torch.float8_e4m3fn), e


def fp8_round(x: torch.Tensor) -> torch.Tensor:
    """float32 values of what 8 bits keep of x's rows (plain torch, any
    device)."""
    q, e = _blocks(x.to(torch.float32))
    q = q.to(torch.float32) * _power_of_two(e).unsqueeze(2)
    return q.flatten(1)[:, :x.shape[1]]


def _operand(x: torch.Tensor, name: str) -> torch.Tensor:
    if not x.is_cuda:
        raise RuntimeError(f"{name}: expected CUDA tensor")
    if x.dtype not in _TYPES:
        raise RuntimeError(f"{name}: expected float32, bfloat16 or float16, "
                           f"got {x.dtype}")
    if x.dim() != 2 or x.shape[0] > _MAX or x.shape[1] > _MAX_INNER:
        raise ValueError(f"{name}: expected a matrix with at most "
                         f"{_MAX_INNER} of the inner dimension and {_MAX} of "
                         f"the other, got shape {tuple(x.shape)}")
    if x.is_neg():                # a sign that torch has put off
        x = x.resolve_neg()
    return x if x.shape[1] <= 1 or x.stride(1) == 1 else x.contiguous()


def _quantise(x: torch.Tensor):
    rows, K = x.shape
    tiles, kb = -(-rows // 16), -(-K // 128)
    q = torch.empty((tiles, kb, 2048), dtype=torch.uint8, device=x.device)
    scales = torch.empty((tiles, -(-kb // 4), 64), dtype=torch.uint8,
                         device=x.device)
    pitch = x.stride(0) if rows > 1 else K
    _launch("ks_fp8_quantise", x.device, x.data_ptr(), _TYPES[x.dtype], pitch,
            rows, K, q.data_ptr(), scales.data_ptr())
    return q, scales


def fp8_pack(W: torch.Tensor) -> Fp8Weight:
    """Quantises a [K, N] weight matrix and lays it out, once."""
    if W.dim() != 2:
        raise ValueError(f"fp8_pack.W: expected a matrix, got shape "
                         f"{tuple(W.shape)}")
    if W.is_cuda:
        _load()
        W = _operand(W.t(), "fp8_pack.W")
        data, scales = _quantise(W)
        return Fp8Weight(data, scales, W.shape[1], W.shape[0])
    K, N = W.shape
    q, e = _blocks(W.t().to(torch.float32))
    tiles, kb = -(-N // 16), e.shape[1]
    q = torch.nn.functional.pad(q.view(torch.uint8),
                                (0, 0, 0, 0, 0, tiles * 16 - N))
    data = q.view(tiles, 16, kb, 2, 2, 4, 8).permute(0, 2, 3, 5, 1, 4, 6) \
        .reshape(tiles, kb, 2048)
    scales = torch.full((tiles * 16, -(-kb // 4) * 4), 127, dtype=torch.uint8)
    scales[:N, :kb] = (e + 127).to(torch.uint8)
    scales = scales.view(tiles, 16, -(-kb // 4), 4).permute(0, 2, 1, 3) \
        .reshape(tiles, -(-kb // 4), 64)
    return Fp8Weight(data.contiguous(), scales.contiguous(), K, N)


def fp8_linear(X: torch.Tensor, W: Fp8Weight,
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``X @ W + bias`` [M, N] in X's type: X's rows are quantised on the
    way, products are summed in float32, the result is rounded once.
    ``bias``: float32 [N].  A float32 result has exact products.  For a 16-bit
    one the matrix unit adds eight neighbours' products at a time and cuts each
    toward zero 2^-13 under the power of two of their largest, so that a result
    is off by up to 7 2^-13 of the largest product of every eight, added up:
    some 1e-5 of the scores' spread where signs are mixed, under 2^-10 of the
    result where all are alike.  Terms that cancel leave it as it is, and it can
    then exceed the result's own rounding."""
    lib = _load()
    X = _operand(X, "fp8_linear.X")
    M, K = X.shape
    if K != W.K:
        raise ValueError(f"fp8_linear: X has {K} columns, W {W.K} rows")
    if W.data.device != X.device or W.scales.device != X.device:
        raise RuntimeError(f"fp8_linear: X is on {X.device}, W on "
                           f"{W.data.device}")
    if bias is not None:
        if bias.device != X.device or bias.dtype != torch.float32:
            raise RuntimeError(f"fp8_linear.bias: expected float32 on "
                               f"{X.device}, got {bias.dtype} on "
                               f"{bias.device}")
        if bias.shape != (W.N,):
            raise ValueError(f"fp8_linear.bias: expected shape ({W.N},), got "
                             f"{tuple(bias.shape)}")
        bias = bias.resolve_neg().contiguous()
    out = X.new_empty((M, W.N))
    if M == 0 or W.N == 0:
        return out
    if K == 0:
        return out.zero_() if bias is None else out.copy_(bias.expand(M, -1))
    kind = _TYPES[X.dtype]
    need = lib.ks_fp8_work(kind, M, K, W.N)
    work = torch.empty(need, dtype=torch.uint8, device=X.device) \
        if need else None
    _launch("ks_fp8_linear", X.device, X.data_ptr(), kind,
            X.stride(0) if M > 1 else K, W.data.data_ptr(),
            W.scales.data_ptr(), _ptr(bias), out.data_ptr(), M, K, W.N,
            _ptr(work))
    return out
