"""A linear classifier on the mean of learned word embeddings.

The mini-batch companion of the n-gram pipelines' LogisticRegression: scores
``S = drop(mean_j E[id_j]) W + b`` with the table E learned along with W,
softmax cross-entropy, synchronous stochastic gradient descent.  A step reads
and writes only the batch's rows of E: the gradient runs along the batch's
sorted tokens, and dropout's mask is drawn again in the backward pass.
"""

from __future__ import annotations

from typing import Optional

import torch

from ...parallel.dataset import TensorDataset
from ...workflow.pipeline import BatchTransformer, LabelEstimator
from ..nlp.embedding import mean_weights, sum_tokens, token_table_grad
from ..stats.dropout import dropout
from .linear import LinearMapper
from .quantized import QuantizedLinearMapper

__all__ = ["EmbeddingClassifierEstimator", "EmbeddingClassifierModel"]


class EmbeddingClassifierModel(BatchTransformer):
    """Word ids [n, L] (-1: no word) to class scores [n, k]."""

    def __init__(self, table: torch.Tensor, head):
        self.table = table
        self.head = head

    def apply_batch(self, ids: torch.Tensor) -> torch.Tensor:
        self.table = self.table.to(ids.device)
        return self.head.apply_batch(sum_tokens(
            self.table, ids, mean_weights(ids, self.table.shape[0],
                                          self.table.dtype)))

    def quantize(self) -> "EmbeddingClassifierModel":
        """The same model with its class weights in 8 bits."""
        return EmbeddingClassifierModel(self.table, self.head.quantize())

    def get_state(self):
        return {"table": self.table,
                **{f"head__{k}": v for k, v in self.head.get_state().items()}}

    def get_config(self):
        return {"quantized": isinstance(self.head, QuantizedLinearMapper),
                "head": self.head.get_config()}

    @classmethod
    def from_saved(cls, config, state):
        head = QuantizedLinearMapper if config["quantized"] else LinearMapper
        return cls(state["table"], head.from_saved(
            config["head"], {k[6:]: v for k, v in state.items()
                             if k.startswith("head__")}))


class EmbeddingClassifierEstimator(LabelEstimator):
    """Fits an EmbeddingClassifierModel on ids [n, L] and integer labels [n].

    Every rank draws its own batches and its own dropout, the gradients are
    summed over all ranks, and all ranks end with the same model.  On one
    rank the table is updated in place, row by row; on several its gradient
    is reduced as a whole."""

    def __init__(self, num_words: int, num_classes: int, dim: int = 64,
                 num_epochs: int = 5, batch_size: int = 256,
                 step_size: float = 1.0, dropout: float = 0.1, seed: int = 0):
        self.num_words = num_words
        self.num_classes = num_classes
        self.dim = dim
        self.num_epochs = num_epochs
        self.batch_size = batch_size
        self.step_size = step_size
        self.dropout = dropout
        self.seed = seed

    def initial(self, device) -> list:
        """[E, W, b], alike on every rank."""
        g = torch.Generator().manual_seed(self.seed)
        E = torch.randn(self.num_words, self.dim, generator=g)
        W = torch.randn(self.dim, self.num_classes, generator=g)
        return [E.to(device), (W / self.dim ** 0.5).to(device),
                torch.zeros(self.num_classes, device=device)]

    def gradients(self, params, ids: torch.Tensor, y: torch.Tensor,
                  total: int, seed: int, step: int,
                  table_rate: Optional[float] = None):
        """The summed cross-entropy of a batch over ``total``, and its
        gradients [dE, dW, db].  With ``table_rate`` dE is None and
        ``table_rate`` times it is added to E."""
        E, W, b = params
        w = mean_weights(ids, E.shape[0], E.dtype)
        h = sum_tokens(E, ids, w)
        hd = dropout(h, self.dropout, seed, step)
        S = hd @ W + b
        logZ = torch.logsumexp(S, dim=1, keepdim=True)
        loss = (logZ - S.gather(1, y.unsqueeze(1))).sum() / total
        dS = torch.exp(S - logZ)
        dS.scatter_add_(1, y.unsqueeze(1), torch.full_like(dS[:, :1], -1.0))
        dS /= total
        dW, db = hd.t() @ dS, dS.sum(0)
        dh = dropout(dS @ W.t(), self.dropout, seed, step)
        if table_rate is None:
            return loss, [token_table_grad(dh, ids, E.shape[0], w), dW, db]
        token_table_grad(dh, ids, E.shape[0], w, table_rate, out=E)
        return loss, [None, dW, db]

    def _fit(self, data: TensorDataset, labels: TensorDataset
             ) -> EmbeddingClassifierModel:
        ids, y, rt = data.data, labels.data, data.runtime
        if y.dim() > 1:
            y = y.argmax(dim=1)
        y = y.to(ids.device).long()
        n, wrong = y.shape[0], None
        if ids.dim() != 2 or ids.shape[0] != n:
            wrong = (f"expected ids [n, L] and labels [n], got "
                     f"{tuple(ids.shape)} and {tuple(y.shape)}")
        elif n and not 0 <= int(y.min()) <= int(y.max()) < self.num_classes:
            wrong = f"expected labels in [0, {self.num_classes})"
        # all ranks refuse what one does: none waits for it in a reduction
        most = torch.tensor([n, wrong is not None], dtype=torch.int64)
        rt.all_reduce_(most, "max")
        if most[1]:
            raise ValueError(wrong or "another rank refused its ids or labels")
        params = self.initial(ids.device)
        steps = self.num_epochs * -(-int(most[0]) // self.batch_size)
        g = torch.Generator().manual_seed(self.seed + 7919 * rt.rank)
        seed = (self.seed + 7919 * rt.rank) % 2 ** 64
        order, at = torch.empty(0, dtype=torch.int64), 0
        for step in range(steps):
            if at >= order.numel():
                order, at = torch.randperm(n, generator=g), 0
            pick = order[at:at + self.batch_size].to(ids.device)
            at += self.batch_size
            if not rt.is_distributed:
                _, grads = self.gradients(params, ids[pick], y[pick],
                                          pick.numel(), seed, step,
                                          -self.step_size)
                for p, d in zip(params[1:], grads[1:]):
                    p -= self.step_size * d
                continue
            _, grads = self.gradients(params, ids[pick], y[pick], 1, seed,
                                      step)
            count = torch.full((1,), float(pick.numel()), device=ids.device)
            rt.all_reduce_many_(grads + [count])
            for p, d in zip(params, grads):
                p -= self.step_size * d / count
        E, W, b = params
        return EmbeddingClassifierModel(E, LinearMapper(W, b))
