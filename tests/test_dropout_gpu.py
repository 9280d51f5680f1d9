"""Dropout from a counter against the generator written out in 64 bits."""

import numpy as np
import pytest
import torch

from tests.philox import expected, philox

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def hip():
    from keystone_amd import hip as h
    assert h.available(), "HIP extension must be built and loadable"
    return h


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9, 1), (33, 65),
                                   (257, 1000), (0, 5), (2, 3, 5)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9999])
def test_dropout(hip, dtype, shape, p):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1))
    x = x.to(dtype).cuda()
    for seed, step in ((0, 0), (2 ** 64 - 1, 2 ** 64 - 1), (12345, 2 ** 33)):
        want, _ = expected(x, p, seed, step)
        assert torch.equal(hip.dropout(x, p, seed, step).cpu(), want)
    if p == 0.0:
        assert torch.equal(hip.dropout(x, p, 3), x)


def test_views_and_in_place(hip):
    base = torch.randn(70, 33, device="cuda")
    for x in (base.t(), base[:, 1:], base[1:], base.view(-1)[1:],
              base[:1].expand(5, 33)):
        want, _ = expected(x, 0.3, 9, 2)
        assert torch.equal(hip.dropout(x, 0.3, 9, 2).cpu(), want)
    want, _ = expected(base, 0.3, 9, 2)
    assert hip.dropout(base, 0.3, 9, 2, out=base) is base
    assert torch.equal(base.cpu(), want)


def test_dropped_places_are_zero_whatever_they_held(hip):
    x = torch.full((1000,), float("nan"), device="cuda")
    _, keep = expected(x, 0.5, 4, 0)
    y = hip.dropout(x, 0.5, 4).cpu()
    assert y[keep].isnan().all() and y[~keep].eq(0).all()


def test_gradient_is_the_same_mask_and_agrees_with_differences(hip):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(100, generator=g).cuda()
    dy = torch.randn(100, generator=g).cuda()
    dx = hip.dropout(dy, 0.25, 5, 7).cpu().double()
    for i in range(100):
        f = []
        for h in (0.5, -0.5):
            z = x.clone()
            z[i] = h                 # exact steps: f is linear in x
            f.append((hip.dropout(z, 0.25, 5, 7).double() * dy).sum().item())
        # one product's rounding in y and one in dx, the sum's in 64 bits
        assert abs(f[0] - f[1] - dx[i]) <= 4 * 2.0 ** -24 * dx[i].abs() + 1e-12


def test_kept_share_and_mean(hip):
    """n = 2^22 fair draws: the kept share is within 6 standard deviations,
    and so is the share of neighbours that are kept together."""
    n = 2 ** 22
    for p in (0.1, 0.5):
        kept = hip.dropout(torch.ones(n, device="cuda"), p, 1, 3) > 0
        q = 1 - round(p * 65536) / 65536
        sd = (q * (1 - q) / n) ** 0.5
        assert abs(kept.double().mean().item() - q) < 6 * sd
        both = (kept[:-1] & kept[1:]).double().mean().item()
        assert abs(both - q * q) < 6 * (3 * q * q * (1 - q * q) / n) ** 0.5


def test_step_on_the_device_in_a_graph(hip):
    x = torch.randn(5000, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        hip.dropout(x, 0.4, 11, step)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hip.dropout(x, 0.4, 11, step)
        step.add_(1)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, hip.dropout(x, 0.4, 11, k))


def test_over_32_bits_of_elements(hip):
    n = 2 ** 32 + 24
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    y = hip.dropout(x, 0.5, 6, out=x)
    tail = y[2 ** 32:].float().cpu()
    b = np.arange(2 ** 29, 2 ** 29 + 3, dtype=np.uint64)
    z = np.zeros_like(b)
    bits = philox(np.stack([b, z, z, z], 1), (6, 0)).view(np.uint16)
    assert torch.equal(tail, torch.from_numpy(
        np.where(bits.reshape(-1) >= 32768, 2.0, 0.0).astype(np.float32)))
