"""Token embeddings on the GPU: lookup, bag sums and the table's gradient.

    embedding_lookup(T, ids, s)            Y[i]  = s T[ids_i]
    embedding_bag(T, ids, offsets, w, s)   Y[b]  = s sum_{j in b} w_j T[ids_j]
    embedding_grad(dY, plan, w, s)         dT[v] = s sum_{ids_j = v} w_j dY[row_j]

An id outside ``[0, V)`` (``WordFrequencyEncoder`` gives an unseen word -1)
reads nothing: a row of zeros, no term of a sum, no gradient.  With CSR
features ``X`` (``crow_indices``, ``col_indices``, ``values`` as offsets, ids
and weights) the bag sum is ``X @ T`` and the gradient ``X.T @ dY``.

Tables and gradients are float32, bfloat16 or float16 with unit inner stride;
sums are held in float32 and rounded once.  Every sum has one order, so two
runs give the same bits.  Nothing is kept for autograd: the gradient is a call.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _launch, _load, _ptr

__all__ = ["EmbeddingPlan", "embedding_lookup", "embedding_bag",
           "embedding_plan", "embedding_grad", "MAX_TOKENS"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MAX_ROWS = 2 ** 31 - 2 ** 16     # of a table that is looked up
MAX_TOKENS = 2 ** 29              # ids, bags and rows of a sum or gradient
_MAX_DIM = 2 ** 22


def _matrix(t: torch.Tensor, name: str) -> torch.Tensor:
    """A readable [rows, D] matrix: unit inner stride, any row pitch."""
    if not t.is_cuda:
        raise RuntimeError(f"{name}: expected CUDA tensor")
    if t.dtype not in _TYPES:
        raise RuntimeError(f"{name}: expected float32, bfloat16 or float16, "
                           f"got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name}: expected a matrix, got shape "
                         f"{tuple(t.shape)}")
    rows, D = t.shape
    if rows > _MAX_ROWS or D > _MAX_DIM:
        raise ValueError(f"{name}: {tuple(t.shape)} is over {_MAX_ROWS} rows "
                         f"or {_MAX_DIM} columns")
    if t.is_neg():                # a sign that torch has put off
        t = t.resolve_neg()
    if D > 1 and t.stride(1) != 1:
        return t.contiguous()
    return t


def _whole(t: torch.Tensor, name: str, device) -> torch.Tensor:
    if t.device != device:
        raise RuntimeError(f"{name}: expected a tensor on {device}, got one "
                           f"on {t.device}")
    if t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{name}: expected int32 or int64, got {t.dtype}")
    return t.contiguous()


def _weights(w: Optional[torch.Tensor], n: int, name: str, device):
    if w is None:
        return None
    if w.device != device or w.dtype != torch.float32:
        raise RuntimeError(f"{name}: expected float32 on {device}, got "
                           f"{w.dtype} on {w.device}")
    if w.numel() != n:
        raise ValueError(f"{name}: {w.numel()} weights for {n} ids")
    if w.is_neg():
        w = w.resolve_neg()
    return w.contiguous()


def _pitch(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _width(D: int, size: int) -> int:
    """Elements of a row that a lane reads at once: a power of two, a row's at
    most and 16 bytes'."""
    return min(1 << D.bit_length() - 1, 16 // size)


def _bags(ids: torch.Tensor, offsets: Optional[torch.Tensor], name: str):
    """(kind, offsets, fixed length, bags) as the kernels take them."""
    if offsets is None:
        return 0, None, int(ids.shape[1]), int(ids.shape[0])
    offsets = _whole(offsets, f"{name}.offsets", ids.device)
    if ids.dim() != 1 or offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError(f"{name}: offsets [bags + 1] go with ids in one "
                         f"dimension, got {tuple(offsets.shape)} and "
                         f"{tuple(ids.shape)}")
    return (1 if offsets.dtype == torch.int32 else 2, offsets, 0,
            offsets.numel() - 1)


def _span(t: torch.Tensor):
    lo = t.data_ptr()
    return lo, lo + ((t.shape[0] - 1) * _pitch(t) + t.shape[1]) * t.element_size()


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor,
                     scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]``: [*ids.shape, D] in the table's type, zeros for
    an id outside the table."""
    lib = _load()
    table = _matrix(table, "embedding_lookup.table")
    ids = _whole(ids, "embedding_lookup.ids", table.device)
    V, D = table.shape
    out = table.new_empty((*ids.shape, D))
    n = ids.numel()
    if n and D:
        _launch("ks_embedding_lookup", table.device, ids.data_ptr(),
                ids.dtype == torch.int64, n, table.data_ptr(),
                _TYPES[table.dtype], V, table.stride(0) if V > 1 else D,
                out.data_ptr(), D, scale, _width(D, table.element_size()))
    return out


def _segment_sum(lib, kind, bounds, fixed, count, n, ids, ids_wide, V, order,
                 weights, keys, src, out, scale, accumulate):
    """V: src's rows, count: out's."""
    D = out.shape[1]
    if count == 0 or D == 0:
        return
    vec = _width(D, src.element_size())
    work = None
    need = lib.ks_segment_work(n, D, vec, keys is not None)
    if need:
        work = src.new_empty(need, dtype=torch.float32)
    _launch("ks_segment_sum", src.device, kind, bounds, fixed, count, n, ids,
            ids_wide, V, order, _ptr(weights), keys, src.data_ptr(),
            _TYPES[src.dtype], src.stride(0) if V > 1 else D, out.data_ptr(),
            _TYPES[out.dtype], out.stride(0) if count > 1 else D, _ptr(work), D,
            scale, accumulate, vec)


def embedding_bag(table: torch.Tensor, ids: torch.Tensor,
                  offsets: Optional[torch.Tensor] = None,
                  weights: Optional[torch.Tensor] = None,
                  scale: float = 1.0) -> torch.Tensor:
    """``Y[b] = scale * sum_j weights_j table[ids_j]`` over the ids of bag b:
    [bags, D] in the table's type, zeros for an empty bag.

    ``offsets`` [bags + 1], ascending, cut ids [n] into bags (ids before the
    first and behind the last belong to none); without them ids are [bags,
    length].  ``weights``: float32, one for each id.  At most 2^29 ids and
    bags."""
    lib = _load()
    table = _matrix(table, "embedding_bag.table")
    ids = _whole(ids, "embedding_bag.ids", table.device)
    if offsets is None and ids.dim() != 2:
        raise ValueError("embedding_bag: without offsets ids are [bags, "
                         f"length], got shape {tuple(ids.shape)}")
    kind, offsets, fixed, bags = _bags(ids, offsets, "embedding_bag")
    n = ids.numel()
    if n > MAX_TOKENS or bags > MAX_TOKENS:
        raise ValueError(f"embedding_bag: {n} ids in {bags} bags are over "
                         f"{MAX_TOKENS}")
    if weights is not None and weights.dim() > 1 \
            and weights.shape != ids.shape:
        raise ValueError(f"embedding_bag.weights: {tuple(weights.shape)} for "
                         f"ids {tuple(ids.shape)}")
    weights = _weights(weights, n, "embedding_bag.weights", table.device)
    V, D = table.shape
    if n == 0:
        return torch.zeros(bags, D, dtype=table.dtype, device=table.device)
    out = table.new_empty((bags, D))
    _segment_sum(lib, kind, _ptr(offsets), fixed, bags, n, ids.data_ptr(),
                 ids.dtype == torch.int64, V, None, weights, None, table, out,
                 scale, False)
    return out


class EmbeddingPlan:
    """Token ids in sorted order: what ``embedding_grad`` sums along.  It
    holds for as long as the ids and the bags do, so a solver that passes
    over the same rows again keeps it.

    ``order`` [n]: positions by ascending token, ascending within a token,
    those outside the table or outside every bag last; ``rows`` [n]: their
    bags (positions themselves where the ids are not pooled); ``keys`` [n]:
    their tokens; ``starts`` [V + 1]: where each token begins."""

    def __init__(self, kept: torch.Tensor, num_rows: int, num_bags: int,
                 n: int, bagged: bool):
        self.num_rows, self.num_bags, self.n = num_rows, num_bags, n
        self.device = kept.device
        # keys, order, rows where there are bags, starts: one allocation
        self._kept, self._bagged = kept, bagged

    def record_stream(self, stream) -> None:
        """As ``torch.Tensor.record_stream``: a plan that is used on another
        stream than the one it was made on and let go of meanwhile keeps its
        memory until that stream is past here."""
        self._kept.record_stream(stream)

    def _places(self):
        """Where keys, order, rows and starts lie."""
        at, step = _ptr(self._kept), 4 * self.n
        rows = at + 2 * step if self._bagged else at + step
        return at, at + step, rows, rows + step

    @property
    def keys(self) -> torch.Tensor:
        return self._kept[:self.n]

    @property
    def order(self) -> torch.Tensor:
        return self._kept[self.n:2 * self.n]

    @property
    def rows(self) -> torch.Tensor:
        return self._kept[2 * self.n:3 * self.n] if self._bagged \
            else self.order

    @property
    def starts(self) -> torch.Tensor:
        return self._kept[self._kept.numel() - self.num_rows - 1:]


def embedding_plan(ids: torch.Tensor, num_rows: int,
                   offsets: Optional[torch.Tensor] = None,
                   pooled: bool = False) -> EmbeddingPlan:
    """Sorts token ids of a table with ``num_rows`` rows.  ``offsets`` as in
    ``embedding_bag``; without them each id is a row of its own
    (``embedding_lookup``), or with ``pooled`` ids are [bags, length]."""
    lib = _load()
    if not ids.is_cuda:
        raise RuntimeError("embedding_plan.ids: expected CUDA tensor")
    ids = _whole(ids, "embedding_plan.ids", ids.device)
    if pooled and offsets is None and ids.dim() != 2:
        raise ValueError("embedding_plan: pooled ids without offsets are "
                         f"[bags, length], got shape {tuple(ids.shape)}")
    n, V = ids.numel(), int(num_rows)
    bagged = pooled or offsets is not None
    kind, fixed, bags = 0, 1, n
    if bagged:
        kind, offsets, fixed, bags = _bags(ids, offsets, "embedding_plan")
    if not 0 <= V <= MAX_TOKENS or n > MAX_TOKENS or bags > MAX_TOKENS:
        raise ValueError(f"embedding_plan: {n} ids in {bags} bags over {V} "
                         f"rows are over {MAX_TOKENS}")
    kept = ids.new_empty((3 if bagged else 2) * n + V + 1, dtype=torch.int32)
    need = lib.ks_token_sort_work(n, V)
    work = ids.new_empty(need, dtype=torch.int32) if need else None
    plan = EmbeddingPlan(kept, V, bags, n, bagged)
    keys, order, rows, starts = plan._places()
    _launch("ks_token_sort", ids.device, ids.data_ptr(),
            ids.dtype == torch.int64, n, V, kind, _ptr(offsets), fixed, bags,
            keys, order, rows if bagged else None, starts, _ptr(work))
    return plan


def embedding_grad(grad: torch.Tensor, plan: EmbeddingPlan,
                   weights: Optional[torch.Tensor] = None, scale: float = 1.0,
                   out: Optional[torch.Tensor] = None,
                   accumulate: bool = False,
                   dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The gradient with respect to the table: [num_rows, D] where row v is
    ``scale`` times the sum of ``weights_j grad[row_j]`` over the occurrences
    of token v, zeros for a token that does not occur.

    ``grad``: [bags, D] of ``embedding_bag`` or [*ids.shape, D] of
    ``embedding_lookup``.  With ``out`` and ``accumulate`` the sums are added
    to ``out``, and rows of tokens that do not occur are left as they are: a
    step of gradient descent is ``embedding_grad(dY, plan, scale=-rate,
    out=table, accumulate=True)``."""
    lib = _load()
    if grad.dim() != 2 and grad.dim():     # rows may have no columns
        grad = grad.reshape(math.prod(grad.shape[:-1]), grad.shape[-1])
    grad = _matrix(grad, "embedding_grad.grad")
    if grad.device != plan.device:
        raise RuntimeError(f"embedding_grad.grad: expected a tensor on "
                           f"{plan.device}, got one on {grad.device}")
    if grad.shape[0] != plan.num_bags:
        raise ValueError(f"embedding_grad: {grad.shape[0]} rows of gradient "
                         f"for a plan of {plan.num_bags}")
    weights = _weights(weights, plan.n, "embedding_grad.weights", grad.device)
    shape = (plan.num_rows, grad.shape[1])
    if out is None:
        if accumulate:
            raise ValueError("embedding_grad: accumulate needs out")
        if dtype not in _TYPES:
            raise RuntimeError(f"embedding_grad: expected float32, bfloat16 "
                               f"or float16, got {dtype}")
        out = grad.new_empty(shape, dtype=dtype)
    else:
        if out.shape != shape:
            raise ValueError(f"embedding_grad.out: expected shape {shape}, "
                             f"got {tuple(out.shape)}")
        if out.dtype not in _TYPES or out.device != grad.device:
            raise RuntimeError(f"embedding_grad.out: expected float32, "
                               f"bfloat16 or float16 on {grad.device}, got "
                               f"{out.dtype} on {out.device}")
        if (out.shape[1] > 1 and out.stride(1) != 1) or \
                (out.shape[0] > 1 and out.stride(0) < out.shape[1]) \
                or out.is_neg():
            raise RuntimeError("embedding_grad.out: rows must be contiguous "
                               "and apart, and no negated view")
        if out.numel() and grad.numel():
            a, b = _span(out)
            read = {"grad": _span(grad)}
            if weights is not None:
                c = weights.data_ptr()
                read["weights"] = c, c + 4 * weights.numel()
            for name, (c, d) in read.items():
                if a < d and c < b:
                    raise ValueError(f"embedding_grad: out overlaps {name}")
    if plan.n == 0 or plan.num_bags == 0:
        return out if accumulate else out.zero_()
    keys, order, rows, starts = plan._places()
    _segment_sum(lib, 1, starts, 0, plan.num_rows, plan.n, rows, 0,
                 plan.num_bags, order, weights, keys, grad, out, scale,
                 accumulate)
    return out
