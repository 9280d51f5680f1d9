"""Linear maps served with 8-bit weights and features.

A fitted LinearMapper or BlockLinearMapper turns into a QuantizedLinearMapper
(``quantize()``), or an estimator of one into ``QuantizedEstimator(est)``.
Weights are quantised once, a row's features on the way; every 128 neighbours
along the features share a power-of-two scale (``keystone_amd.hip.fp8``).
Scores are off by a few hundredths of their terms' spread: for ranking
classes, not for solving.
"""

from __future__ import annotations

from typing import Optional

import torch

from ...parallel.dataset import Dataset, TensorDataset
from ...utils.derivatives import differentiated
from ...workflow.pipeline import (BatchTransformer, LabelEstimator,
                                  TupleDataset)

__all__ = ["QuantizedLinearMapper", "QuantizedEstimator"]


class QuantizedLinearMapper(BatchTransformer):
    """``x -> x W + b`` with e4m3 operands (stands in for LinearMapper and
    BlockLinearMapper on the serving path)."""

    def __init__(self, packed, b: Optional[torch.Tensor] = None):
        self.packed = packed
        self.b = None if b is None else b.to(torch.float32)

    @classmethod
    def from_weights(cls, W: torch.Tensor, b: Optional[torch.Tensor] = None):
        from ... import hip
        if W.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            W = W.to(torch.float32)
        return cls(hip.fp8_pack(W), b)

    def apply_batch(self, X: torch.Tensor) -> torch.Tensor:
        if X.dim() < 2 or X.shape[-1] != self.packed.K:
            raise ValueError(f"QuantizedLinearMapper: rows {tuple(X.shape)} of "
                             f"features for {self.packed.K} weights")
        if X.dim() == 2:
            return self._rows(X)
        out = self._rows(X.reshape(X.shape[:-1].numel(), X.shape[-1]))
        return out.reshape(*X.shape[:-1], self.packed.N)

    def _rows(self, X: torch.Tensor) -> torch.Tensor:
        from ... import hip
        if self.packed.data.device != X.device:
            self.packed = self.packed.to(X.device)
        if self.b is not None:
            self.b = self.b.to(X.device)
        # what the kernel returns has no gradient; torch's rounding passes it on
        if X.is_cuda and not differentiated(X, self.b) and hip.gpu_ready():
            if X.dtype in (torch.float32, torch.bfloat16, torch.float16):
                return hip.fp8_linear(X, self.packed, self.b)
            out = hip.fp8_linear(X.to(torch.float32), self.packed, self.b)
        else:
            out = hip.fp8_round(X) @ self.packed.dequantise()
            if self.b is not None:
                out = out + self.b
        # whole numbers' scores are none
        return out.to(X.dtype) if X.is_floating_point() else out

    def apply(self, x):
        if isinstance(x, (tuple, list)):
            x = torch.cat(list(x), dim=-1)
        if x.dim() > 1:
            return self.apply_batch(x)
        return self.apply_batch(x.unsqueeze(0)).squeeze(0)

    def apply_dataset(self, ds: Dataset) -> Dataset:
        if isinstance(ds, TupleDataset):   # VectorSplitter's blocks
            return TensorDataset(self.apply_batch(
                torch.cat([p.data for p in ds.parts], dim=-1)), ds.runtime)
        return super().apply_dataset(ds)

    def get_state(self):
        st = {"data": self.packed.data, "scales": self.packed.scales}
        if self.b is not None:
            st["b"] = self.b
        return st

    def get_config(self):
        return {"K": self.packed.K, "N": self.packed.N}

    @classmethod
    def from_saved(cls, config, state):
        from ... import hip
        return cls(hip.Fp8Weight(state["data"], state["scales"], config["K"],
                                 config["N"]), state.get("b"))


class QuantizedEstimator(LabelEstimator):
    """Fits ``inner`` and quantises the linear map that it gives."""

    def __init__(self, inner: LabelEstimator):
        from ...workflow.state_cache import _estimator_key
        self.inner = inner
        # names the inner estimator where fitted state is looked up by what
        # an estimator's plain attributes hold
        self.inner_key = _estimator_key(inner)

    def _fit(self, data: Dataset, labels: Dataset) -> QuantizedLinearMapper:
        fitted = self.inner._fit(data, labels)
        if not hasattr(fitted, "quantize"):
            raise TypeError(f"QuantizedEstimator: {type(fitted).__name__} is "
                            "no linear map")
        return fitted.quantize()
