"""The token, dropout and 8-bit operators at their edges, on the CPU."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from keystone_amd.utils.derivatives import differentiated


def test_what_counts_as_differentiated():
    x, r = torch.ones(3), torch.ones(3, requires_grad=True)
    assert not differentiated(x, None) and differentiated(None, x, r)
    with torch.no_grad():
        assert not differentiated(r)
    seen = []

    def f(t):
        seen.append(differentiated(t))
        return t.sum()

    torch.func.vmap(f)(torch.ones(2, 3))
    torch.func.jvp(f, (x,), (x,))
    torch.func.grad(f)(x)
    assert seen == [True] * 3
    with fwd.dual_level():
        assert differentiated(fwd.make_dual(x, x)) and not differentiated(x)
    assert not differentiated(x)
