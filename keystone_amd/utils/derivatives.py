"""Whether torch is asked for a derivative of a call.

The HIP kernels read memory and keep nothing for autograd, so calls that are
differentiated go through plain torch instead.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.autograd.forward_ad as _forward

__all__ = ["differentiated"]


def differentiated(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether one of them asks for its gradient, has a tangent (forward
    mode, which leaves ``requires_grad`` alone) or stands for another tensor
    inside a transform of ``torch.func``."""
    reverse = torch.is_grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if reverse and t.requires_grad:
            return True
        if torch._C._functorch.is_functorch_wrapped_tensor(t):
            return True
        if _forward._current_level >= 0 and \
                _forward.unpack_dual(t).tangent is not None:
            return True
    return False
