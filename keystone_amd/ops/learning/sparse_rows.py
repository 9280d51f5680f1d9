"""CSR rows as the iterative solvers multiply by them on the GPU.

With a row's column indices as the tokens of a bag and its values as their
weights, ``X @ W`` is a sum of W's rows over bags and ``X.T @ D`` the gradient
of such a sum, by columns sorted once for the whole fit.  An intercept is a
column of ones that is never stored.
"""

from __future__ import annotations

import torch

from ...utils.derivatives import differentiated

__all__ = ["SparseRows", "csr_matmul"]


def csr_matmul(X: torch.Tensor, W: torch.Tensor) -> torch.Tensor:
    """``X @ W`` of CSR rows that ``SparseRows.supports``."""
    # the kernels keep nothing for autograd, and take no shape that does not fit
    if W.dim() != 2 or differentiated(W):
        return X @ W
    if X.shape[1] != W.shape[0]:
        raise RuntimeError(f"rows of {X.shape[1]} features by weights "
                           f"{tuple(W.shape)}")
    from ... import hip
    return hip.embedding_bag(W, X.col_indices(), X.crow_indices(), X.values())


class SparseRows:
    """float32 CSR rows [n, d] on the GPU, with ``intercept`` [n, d + 1]."""

    def __init__(self, csr: torch.Tensor, intercept: bool = False):
        from ... import hip
        self.hip = hip
        self.offsets = csr.crow_indices()
        self.columns = csr.col_indices()
        self.values = csr.values()
        self.intercept = intercept
        self.features = csr.shape[1]
        self.shape = torch.Size((csr.shape[0], csr.shape[1] + intercept))
        self.plan = hip.embedding_plan(self.columns, self.features,
                                       self.offsets)

    @staticmethod
    def supports(X: torch.Tensor) -> bool:
        """Whether X is such rows, with sizes that the kernels take."""
        if not (X.layout == torch.sparse_csr and X.is_cuda
                and X.dtype == torch.float32 and X.dim() == 2):
            return False
        if X.requires_grad and torch.is_grad_enabled():
            return False
        from ... import hip
        return max(*X.shape, X.values().numel()) <= hip.MAX_TOKENS \
            and hip.gpu_ready()

    @staticmethod
    def mostly_filled(X: torch.Tensor) -> bool:
        """Whether so many of X's entries are stored that its products are
        faster dense.  ``X @ W`` and ``X.T @ D`` of 20000 x 20000 by 20
        columns take 0.57 ms here with 5 in 100 stored, 1.2 ms with 10, and
        0.70 ms dense; by 147 columns 3.1, 6.1 and 2.7 ms."""
        return X.values().numel() * 16 > X.shape[0] * X.shape[1]

    def __matmul__(self, W: torch.Tensor) -> torch.Tensor:
        S = self.hip.embedding_bag(W[:self.features], self.columns,
                                   self.offsets, self.values)
        return S + W[self.features] if self.intercept else S

    def t_matmul(self, D: torch.Tensor) -> torch.Tensor:
        """``X.T @ D``."""
        out = torch.empty(self.shape[1], D.shape[1], dtype=torch.float32,
                          device=D.device)
        self.hip.embedding_grad(D, self.plan, self.values,
                                out=out[:self.features])
        if self.intercept:
            out[self.features] = D.sum(0)
        return out
