"""Token lookup, bag sums and the table's gradient against 64-bit sums.

A sum of m products in float32 is off by at most (m + 2) 2^-24 of the sum of
their magnitudes (one rounding a term, one by the scale), and the result's
rounding by half a step of its type."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def hip():
    from keystone_amd import hip as h
    assert h.available(), "HIP extension must be built and loadable"
    return h


def gen(seed):
    return torch.Generator().manual_seed(seed)


def some_ids(n, V, g, hot=0.3, unseen=0.1, wide=True):
    """Ids with one hot token and some outside the table on both sides."""
    ids = torch.randint(0, max(V, 1), (n,), generator=g)
    u = torch.rand(n, generator=g)
    ids = torch.where(u < hot, torch.full_like(ids, V // 2), ids)
    ids = torch.where(u > 1 - unseen / 2, torch.full_like(ids, -1), ids)
    ids = torch.where((u > 1 - unseen) & (u <= 1 - unseen / 2),
                      torch.full_like(ids, V), ids)
    return (ids if wide else ids.int()).cuda()


def some_offsets(lens, wide=True):
    o = torch.zeros(len(lens) + 1, dtype=torch.int64)
    o[1:] = torch.cumsum(torch.tensor(lens, dtype=torch.int64), 0)
    return (o if wide else o.int()).cuda()


def sums64(src, rows, dst, weights, count, scale):
    """scale * sum of weights * src[rows] into dst, the magnitudes' sum and
    the number of terms, in 64 bits on the CPU; rows or dst of -1: no term."""
    rows, dst = rows.cpu().long(), dst.cpu().long()
    w = torch.ones(rows.numel(), dtype=torch.float64) if weights is None \
        else weights.cpu().double()
    ok = (rows >= 0) & (rows < src.shape[0]) & (dst >= 0) & (dst < count)
    v = src.cpu().double()[rows[ok]] * (w[ok] * scale)[:, None]
    z = torch.zeros(count, src.shape[1], dtype=torch.float64)
    m = torch.bincount(dst[ok], minlength=count).double()[:, None]
    return (z.index_add(0, dst[ok], v), z.index_add(0, dst[ok], v.abs()), m)


def check(got, want, mag, m):
    i = torch.finfo(got.dtype)
    tol = (m + 2) * 2.0 ** -24 * mag + i.eps / 2 * want.abs() \
        + i.tiny * i.eps / 2
    off = (got.cpu().double() - want).abs() - tol * (1 + 1e-9)
    assert off.max() <= 0 if off.numel() else True, off.max()


def bag_of(offsets, n):
    o = offsets.cpu().long()
    return torch.searchsorted(o, torch.arange(n), right=True) - 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,V,D", [
    ((1,), 1, 1), ((7,), 3, 5), ((5, 13), 50, 64), ((1000,), 777, 100),
    ((257,), 20000, 1030), ((3, 0), 9, 8), ((33,), 7, 300), ((9,), 4, 0)])
def test_lookup(hip, dtype, shape, V, D):
    g = gen(V * 31 + D)
    table = torch.randn(V, D, generator=g).to(dtype).cuda()
    n = math.prod(shape)
    ids = some_ids(n, V, g, wide=D % 2 == 0).view(shape)
    for scale in (1.0, 3.7):
        got = hip.embedding_lookup(table, ids, scale)
        assert got.shape == (*shape, D) and got.dtype == dtype
        flat = ids.reshape(-1)
        want, mag, m = sums64(table, flat, torch.arange(n), None, n, scale)
        check(got.view(n, D), want, mag, m)


def test_lookup_strided_and_misaligned_tables(hip):
    g = gen(1)
    base = torch.randn(40, 71, generator=g).cuda()
    ids = some_ids(64, 40, g)
    for t in (base[:, 3:67], base[:, :64], base[::2], base.t(),
              base[:1].expand(40, 71), base.view(-1)[1:1 + 39 * 71].view(39, 71)):
        ok = ids.clone()
        ok[ids >= t.shape[0]] = -1
        want = torch.where((ok >= 0)[:, None], t[ok.clamp(min=0)],
                           torch.zeros((), device="cuda"))
        assert torch.equal(hip.embedding_lookup(t, ids), want)


def test_absent_rows_are_not_read_into_the_sum(hip):
    table = torch.full((4, 8), float("nan"), device="cuda")
    ids = torch.tensor([[-1, 4], [2 ** 40, -2 ** 40]], device="cuda")
    assert torch.equal(hip.embedding_lookup(table, ids),
                       torch.zeros(2, 2, 8, device="cuda"))
    assert torch.equal(hip.embedding_bag(table, ids),
                       torch.zeros(2, 8, device="cuda"))


LENGTHS = {
    "empty_all": [0, 0, 0], "one": [1], "ones": [1] * 70,
    "empty_between": [0, 3, 0, 0, 5, 1, 0],
    "border": [127, 128, 129, 0, 256, 1, 255],
    "one_long": [5000], "long_between": [3, 1000, 0, 0, 130, 2, 4000, 7],
    "many": [(7 * i) % 41 for i in range(600)],
}


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 2, 20, 63, 256, 520])
def test_bag(hip, dtype, lens, D):
    lens = LENGTHS[lens]
    n, g = sum(lens), gen(D + len(lens))
    V = 97
    table = torch.randn(V, D, generator=g).to(dtype).cuda()
    ids = some_ids(n, V, g, wide=D % 2 == 0)
    offsets = some_offsets(lens, wide=D % 3 != 0)
    for weights, scale in ((None, 1.0),
                           (torch.randn(n, generator=g).cuda(), 0.3)):
        got = hip.embedding_bag(table, ids, offsets, weights, scale)
        assert got.shape == (len(lens), D) and got.dtype == dtype
        check(got, *sums64(table, ids, bag_of(offsets, n), weights, len(lens),
                           scale))
        again = hip.embedding_bag(table, ids, offsets, weights, scale)
        assert torch.equal(got, again)


@pytest.mark.parametrize("B,L", [(1, 1), (5, 0), (0, 4), (3, 129), (2, 2000),
                                 (400, 9)])
def test_bag_of_fixed_length(hip, B, L):
    g = gen(B + L)
    table = torch.randn(50, 36, generator=g).cuda()
    ids = some_ids(B * L, 50, g).view(B, L)
    w = torch.rand(B, L, generator=g).cuda()
    got = hip.embedding_bag(table, ids, weights=w)
    bag = torch.arange(B * L) // max(L, 1)
    check(got, *sums64(table, ids.reshape(-1), bag, w.reshape(-1), B, 1.0))


def test_ids_outside_every_bag_are_left_out(hip):
    table = torch.eye(4, device="cuda")
    ids = torch.tensor([0, 1, 2, 3, 0, 1], device="cuda")
    offsets = torch.tensor([1, 3, 4], device="cuda")
    want = torch.tensor([[0., 1, 1, 0], [0, 0, 0, 1]], device="cuda")
    assert torch.equal(hip.embedding_bag(table, ids, offsets), want)
    plan = hip.embedding_plan(ids, 4, offsets)
    dy = torch.tensor([[1., 2], [10, 20]], device="cuda")
    want = torch.tensor([[0., 0], [1, 2], [1, 2], [10, 20]], device="cuda")
    assert torch.equal(hip.embedding_grad(dy, plan), want)


@pytest.mark.parametrize("n,V", [
    (n, V) for V in (0, 1, 2, 255, 511, 512, 5000, 300000)
    for n in (0, 1, 63, 4095, 4097, 20011)] + [(4097, 2 ** 27),
                                               (9001, 2 ** 27)])
def test_plan_is_a_stable_sort(hip, n, V):
    g = gen(n + V)
    ids = some_ids(n, V, g, wide=n % 2 == 0)
    p = hip.embedding_plan(ids, V)
    key = torch.where((ids >= 0) & (ids < V), ids, torch.full_like(ids, V))
    want, order = torch.sort(key.cpu().long(), stable=True)
    assert torch.equal(p.keys.cpu().long(), want)
    assert torch.equal(p.order.cpu().long(), order)
    starts = torch.searchsorted(want, torch.arange(V + 1))
    assert torch.equal(p.starts.cpu().long(), starts)


@pytest.mark.parametrize("V", [1, 2047, 2048, 100001])
@pytest.mark.parametrize("n", [17, 4000, 8191, 8192, 8193, 70001, 262144,
                               262145, 400001, 524288, 524289])
@pytest.mark.parametrize("bags", ["most of them empty", "long", "one", "ten",
                                  "all empty", "fixed"])
def test_plan_of_bags(hip, n, V, bags):
    g = gen(n + V)
    ids = some_ids(n, V, g, wide=n % 2 == 0)
    if bags == "fixed":
        n -= n % 3
        ids = ids[:n].view(-1, 3)
        p = hip.embedding_plan(ids, V, pooled=True)
        bag, ids = torch.arange(n) // 3, ids.reshape(-1)
    else:
        # the first and the last few ids are in no bag
        lo, hi = 3, n - 5
        count = {"most of them empty": 3 * n, "long": 7, "one": 1,
                 "ten": n // 10, "all empty": 1000}[bags]
        at = torch.randint(lo, hi + 1, (count + 1,), generator=g).sort()[0]
        if bags == "all empty":
            at[:] = n // 2
        else:
            at[0], at[-1] = lo, hi
        if bags == "most of them empty":
            at[count // 3:2 * count // 3] = at[count // 3].clone()
            at = at.sort()[0]
        offsets = (at if n % 2 else at.int()).cuda()
        p = hip.embedding_plan(ids, V, offsets)
        i = torch.arange(n)
        bag = torch.searchsorted(at, i, right=True) - 1
        bag = torch.where((i < at[0]) | (i >= at[-1]), -1, bag)
    ids = ids.cpu().long()
    key = torch.where((ids >= 0) & (ids < V) & (bag >= 0), ids, V)
    want, order = torch.sort(key, stable=True)
    assert torch.equal(p.keys.cpu().long(), want)
    assert torch.equal(p.order.cpu().long(), order)
    assert torch.equal(p.starts.cpu().long(),
                       torch.searchsorted(want, torch.arange(V + 1)))
    there, rows = want < V, p.rows.cpu().long()
    assert torch.equal(rows[there], bag[order][there])
    assert rows.min() >= 0 and rows.max() < p.num_bags


@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (50, 7, 33), (777, 2000, 100),
                                   (5000, 3, 260), (9000, 40, 2)])
def test_grad_of_lookup(hip, src, out, n, V, D):
    g = gen(n + D)
    ids = some_ids(n, V, g)
    dy = torch.randn(n, D, generator=g).to(src).cuda()
    plan = hip.embedding_plan(ids, V)
    got = hip.embedding_grad(dy, plan, scale=0.7, dtype=out)
    assert got.dtype == out
    check(got, *sums64(dy, torch.arange(n), ids, None, V, 0.7))
    assert torch.equal(got, hip.embedding_grad(
        dy, hip.embedding_plan(ids, V), scale=0.7, dtype=out))


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("D", [1, 2, 20, 256])
def test_grad_of_bag(hip, lens, D):
    lens = LENGTHS[lens]
    n, g = sum(lens), gen(D)
    V = 61
    ids, offsets = some_ids(n, V, g), some_offsets(lens)
    w = torch.randn(n, generator=g).cuda()
    dy = torch.randn(len(lens), D, generator=g).cuda()
    plan = hip.embedding_plan(ids, V, offsets)
    got = hip.embedding_grad(dy, plan, w, 1.5)
    check(got, *sums64(dy, bag_of(offsets, n), ids, w, V, 1.5))


def test_grad_accumulates_into_the_rows_that_occur(hip):
    g = gen(3)
    V, D, n = 500, 37, 2000
    ids = torch.randint(0, 50, (n,), generator=g).cuda()
    ids[:600] = 7
    dy = torch.randn(n, D, generator=g).cuda()
    flat = torch.randn(V, 64, generator=g).cuda()
    flat[100] = float("nan")
    table = flat[:, 5:5 + D]
    before = flat.clone()
    got = hip.embedding_grad(dy, hip.embedding_plan(ids, V), scale=-0.1,
                             out=table, accumulate=True)
    assert got is table
    want, mag, m = sums64(dy, torch.arange(n), ids, None, V, -0.1)
    seen = before[:50, 5:5 + D].cpu().double()
    check(table[:50], want[:50] + seen, mag[:50] + seen.abs(), m[:50] + 2)
    flat, before = flat.view(torch.int32), before.view(torch.int32)
    assert torch.equal(flat[50:], before[50:])
    assert torch.equal(flat[:, :5], before[:, :5])
    assert torch.equal(flat[:, 5 + D:], before[:, 5 + D:])


def test_grad_agrees_with_differences(hip):
    """d/dT of f(T) = sum(Y * dY) by central differences: f is linear in T,
    so that a difference over 2h is off only by the roundings of Y, half a
    step of float32 sums of at most 6 terms of magnitude below 4."""
    g = gen(5)
    V, D = 6, 4
    ids = torch.tensor([[1, 1, 3], [0, -1, 1]], device="cuda")
    w = torch.rand(2, 3, generator=g).cuda()
    T = torch.rand(V, D, generator=g).cuda()
    dy = torch.rand(2, D, generator=g).cuda()
    plan = hip.embedding_plan(ids, V, pooled=True)
    got = hip.embedding_grad(dy, plan, w, 0.5)
    h = 0.25
    for v in range(V):
        for d in range(D):
            f = []
            for s in (h, -h):
                P = T.clone()
                P[v, d] += s
                y = hip.embedding_bag(P, ids, weights=w, scale=0.5)
                f.append((y.double() * dy.double()).sum().item())
            assert abs((f[0] - f[1]) / (2 * h) - got[v, d].item()) \
                <= 2 * 24 * 2.0 ** -24 * 4 / h


def test_dtype_limits_and_infinities(hip):
    """An infinity goes where its token goes and nowhere else."""
    dy = torch.ones(300, 8, device="cuda")
    dy[17] = float("inf")
    ids = torch.arange(300, device="cuda") % 5
    got = hip.embedding_grad(dy, hip.embedding_plan(ids, 9))
    assert got[2].isinf().all() and got[[0, 1, 3, 4]].eq(60).all()
    assert got[5:].eq(0).all()


def test_a_copied_plan_outlives_the_first(hip):
    import copy
    g = gen(8)
    ids, dy = some_ids(900, 40, g), torch.randn(900, 24, generator=g).cuda()
    plan = hip.embedding_plan(ids, 40)
    want = hip.embedding_grad(dy, plan)
    again = copy.deepcopy(plan)
    assert again.starts.data_ptr() != plan.starts.data_ptr()
    del plan
    torch.zeros(3000, dtype=torch.int32, device="cuda").fill_(-1)
    assert torch.equal(hip.embedding_grad(dy, again), want)


def test_captured_and_replayed(hip):
    """Lookup, plan and gradient in one graph, replayed on changed inputs."""
    g = gen(6)
    V, D, n = 900, 48, 7000
    ids = some_ids(n, V, g)
    T = torch.randn(V, D, generator=g).cuda()
    dy = torch.randn(n, D, generator=g).cuda()

    def step():
        y = hip.embedding_lookup(T, ids, 2.0)
        return y, hip.embedding_grad(dy, hip.embedding_plan(ids, V))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dT = step()
    for k in range(4):
        ids.copy_(some_ids(n, V, g, hot=0.2 * k))
        dy.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        ey, edT = step()
        torch.cuda.synchronize()
        assert torch.equal(y, ey) and torch.equal(dT, edT)


def test_large_table_passes_32_bit_offsets(hip):
    V, D = 2 ** 22 + 3, 520          # 2.2e9 elements
    table = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    table[V - 1] = 3.0
    ids = torch.tensor([V - 1, 0, V - 1], device="cuda")
    got = hip.embedding_lookup(table, ids)
    assert got[0].eq(3).all() and got[1].eq(0).all()
    assert hip.embedding_bag(table, ids[None]).eq(6).all()
    dy = torch.ones(3, D, dtype=torch.bfloat16, device="cuda")
    hip.embedding_grad(dy, hip.embedding_plan(ids, V), out=table,
                       accumulate=True)
    assert table[V - 1].eq(5).all() and table[0].eq(1).all()
    assert table[1:V - 1].count_nonzero() == 0
