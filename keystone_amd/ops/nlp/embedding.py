"""Token embeddings: rows of a table by word id, and their means.

The ids are WordFrequencyEncoder's frequency ranks (ref:
nodes.nlp.WordFrequencyEncoder), -1 for an unseen word.  An id outside the
table stands for no word: zeros from a lookup, no term of a mean, no
gradient.  On the GPU these run as the kernels of ``keystone_amd.hip``, which
keep nothing for autograd: solvers call ``token_table_grad``.  Where a table or
weights are differentiated it is plain torch, as on the CPU.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from ...parallel.dataset import Dataset, TensorDataset
from ...utils.derivatives import differentiated
from ...workflow.pipeline import BatchTransformer, Transformer

__all__ = ["PadTokens", "TokenEmbedding", "MeanEmbedding", "embed_tokens",
           "sum_tokens", "token_table_grad", "mean_weights"]


def _hip(t: torch.Tensor, *others: Optional[torch.Tensor]):
    """The kernels, where t's device and type go through them."""
    if differentiated(t, *others):
        return None
    if t.is_cuda and t.dtype in (torch.float32, torch.bfloat16,
                                 torch.float16):
        from ... import hip
        if hip.gpu_ready():
            return hip
    return None


def _seen(ids: torch.Tensor, rows: int) -> torch.Tensor:
    return (ids >= 0) & (ids < rows)


def _kernel_ids(ids: torch.Tensor) -> torch.Tensor:
    """Ids in one of the kernels' two types."""
    if ids.dtype in (torch.int32, torch.int64) or ids.is_floating_point():
        return ids
    return ids.long()


def _kernel_weights(weights: Optional[torch.Tensor]):
    return None if weights is None else weights.to(torch.float32)


def _bag_weights(weights: Optional[torch.Tensor], ids: torch.Tensor):
    """A weight for each of the ids, that are rows of bags."""
    if ids.dim() != 2:
        raise ValueError(f"expected ids [bags, length], got {tuple(ids.shape)}")
    return None if weights is None else weights.expand(ids.shape)


def _wide(dtype: torch.dtype) -> torch.dtype:
    """What sums are held in: 32 bits or more."""
    return torch.promote_types(dtype, torch.float32)


def embed_tokens(table: torch.Tensor, ids: torch.Tensor,
                 scale: float = 1.0) -> torch.Tensor:
    """``scale * table[ids]``, [*ids.shape, D]."""
    hip = _hip(table, ids)
    if hip is not None:
        return hip.embedding_lookup(table, _kernel_ids(ids), scale)
    seen = _seen(ids, table.shape[0])
    out = table.new_zeros(*ids.shape, table.shape[1])
    out[seen] = table[ids[seen].long()] * scale
    return out


def sum_tokens(table: torch.Tensor, ids: torch.Tensor,
               weights: Optional[torch.Tensor] = None,
               scale: float = 1.0) -> torch.Tensor:
    """``scale * sum_j weights[b, j] table[ids[b, j]]``, [B, D], of ids
    [B, L], in the table's type: rounded once."""
    weights = _bag_weights(weights, ids)
    hip = _hip(table, ids, weights)
    if hip is not None:
        return hip.embedding_bag(table, _kernel_ids(ids), None,
                                 _kernel_weights(weights), scale)
    rows = embed_tokens(table, ids).to(_wide(table.dtype))
    if weights is not None:
        # an absent word's may be a NaN
        weights = weights.masked_fill(~_seen(ids, table.shape[0]), 0.0)
        rows = rows * weights.unsqueeze(-1).to(rows.dtype)
    return (rows.sum(1) * scale).to(table.dtype)


def token_table_grad(grad: torch.Tensor, ids: torch.Tensor, num_rows: int,
                     weights: Optional[torch.Tensor] = None,
                     scale: float = 1.0, out: Optional[torch.Tensor] = None
                     ) -> torch.Tensor:
    """``sum_tokens``'s gradient with respect to the table, [num_rows, D] in
    grad's type; with ``out`` it is added to ``out``."""
    weights = _bag_weights(weights, ids)
    hip = _hip(grad, ids, weights)
    if hip is not None and (out is None or out.dtype in (
            torch.float32, torch.bfloat16, torch.float16)):
        plan = hip.embedding_plan(_kernel_ids(ids), num_rows, pooled=True)
        return hip.embedding_grad(grad, plan, _kernel_weights(weights), scale,
                                  out=out, accumulate=out is not None,
                                  dtype=grad.dtype)
    wide = _wide(grad.dtype)
    g = grad.to(wide).unsqueeze(1).expand(*ids.shape, grad.shape[1])
    seen = _seen(ids, num_rows)
    if weights is not None:
        g = g * weights.masked_fill(~seen, 0.0).unsqueeze(-1).to(wide)
    at, g = ids[seen].long(), g[seen] * scale
    if out is not None and out.dtype == wide:
        return out.index_add_(0, at, g)
    sums = g.new_zeros(num_rows, grad.shape[1]).index_add_(0, at, g)
    return sums.to(grad.dtype) if out is None else out.add_(sums)


def mean_weights(ids: torch.Tensor, num_rows: int,
                 dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[B, L] in 32 bits or more: one over the number of row b's words, so that
    the weighted sum is their mean (zero for a row without any)."""
    n = _seen(ids, num_rows).sum(1, keepdim=True).clamp(min=1)
    return (1.0 / n.to(_wide(dtype))).expand(ids.shape).contiguous()


class PadTokens(Transformer):
    """Word ids of a document to one fixed length: cut off after it, filled
    up with -1."""

    def __init__(self, length: int):
        if length < 1:
            raise ValueError(f"PadTokens: expected a length of at least 1, "
                             f"got {length}")
        self.length = length

    def apply(self, ids: Sequence[int]) -> torch.Tensor:
        ids = list(ids)[:self.length]
        return torch.tensor(ids + [-1] * (self.length - len(ids)),
                            dtype=torch.int64)

    def apply_dataset(self, ds: Dataset) -> TensorDataset:
        rows = [self.apply(x) for x in ds.items()]
        data = torch.stack(rows) if rows else \
            torch.empty(0, self.length, dtype=torch.int64)
        return TensorDataset(data.to(ds.runtime.device), ds.runtime)


class _TableTransformer(BatchTransformer):
    def __init__(self, table: torch.Tensor, scale: float = 1.0):
        if table.dim() != 2 or not table.is_floating_point():
            raise ValueError("expected a floating-point table [words, dim], "
                             f"got {tuple(table.shape)} {table.dtype}")
        self.table = table
        self.scale = scale

    def _resident(self, ids: torch.Tensor) -> torch.Tensor:
        self.table = self.table.to(ids.device)
        return self.table

    @classmethod
    def from_saved(cls, config, state):
        return cls(state["table"], config["scale"])


class TokenEmbedding(_TableTransformer):
    """Word ids [..., L] to their rows of the table, scaled: [..., L, D]."""

    def apply_batch(self, ids: torch.Tensor) -> torch.Tensor:
        return embed_tokens(self._resident(ids), ids, self.scale)


class MeanEmbedding(_TableTransformer):
    """Word ids [n, L] to the mean of their rows of the table, scaled:
    [n, D].  Unseen words (and PadTokens' filling) do not count."""

    def apply_batch(self, ids: torch.Tensor) -> torch.Tensor:
        table = self._resident(ids)
        return sum_tokens(table, ids, mean_weights(ids, table.shape[0],
                                                   table.dtype), self.scale)
