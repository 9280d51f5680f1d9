"""The token, dropout and 8-bit operators on the GPU at their edges: shapes,
types and transforms that the CPU path takes and the kernels' path has to take
alike, and sizes that reach the kernels' large and in-place variants."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import keystone_amd as ka
from keystone_amd.ops.learning import (DenseLBFGSwithL2, LeastSquaresGradient,
                                       LinearMapper, SparseLBFGSwithL2)
from keystone_amd.ops.learning.sparse_rows import SparseRows, csr_matmul
from keystone_amd.ops.nlp.embedding import (embed_tokens, sum_tokens,
                                            token_table_grad)
from keystone_amd.ops.stats import dropout
from tests.test_embedding_gpu import check, gen, some_ids, some_offsets, sums64

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def hip():
    from keystone_amd import hip as h
    assert h.available(), "HIP extension must be built and loadable"
    return h


# ------------------------------------------------------------- 8-bit mapper
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.uint8])
def test_quantized_scores_of_whole_number_features(dtype):
    """Counts as features: the scores are numbers with fractions, as on the
    CPU, and not cut to whole ones."""
    g = gen(1)
    X = torch.randint(0, 9, (20, 200), generator=g).to(dtype)
    q = LinearMapper(torch.randn(200, 7, generator=g),
                     torch.randn(7, generator=g)).quantize()
    want = q.apply_batch(X)
    got = q.apply_batch(X.cuda())
    assert got.dtype == want.dtype == torch.float32
    # 202 roundings of sums of 200 products of at most 8 by 4
    assert torch.allclose(got.cpu(), want, rtol=0, atol=202 * 2 ** -24 * 6400)


def test_quantized_scores_keep_gradients():
    g = gen(2)
    q = LinearMapper(torch.randn(300, 5, generator=g)).quantize()
    X = torch.randn(9, 300, generator=g)
    grads = []
    for x in (X.clone().requires_grad_(), X.cuda().requires_grad_()):
        q.apply_batch(x).square().sum().backward()
        grads.append(x.grad.cpu())
    assert grads[0].abs().sum() > 0
    assert torch.allclose(*grads, rtol=1e-4, atol=1e-4)
    with fwd.dual_level():
        x = fwd.make_dual(X.cuda(), torch.ones(9, 300, device="cuda"))
        assert fwd.unpack_dual(q.apply_batch(x)).tangent is not None


@pytest.mark.parametrize("M,K,N", [(3, 2000, 40), (1100, 2300, 40),
                                   (2100, 2176, 1030)])
def test_packed_weights_from_a_larger_buffer(hip, M, K, N):
    g = gen(K)
    W = hip.fp8_pack(torch.randn(K, N, generator=g).cuda())
    X = torch.randn(M, K, generator=g).cuda()
    buffer = torch.cat([torch.zeros(5, dtype=torch.uint8, device="cuda"),
                        W.data.reshape(-1), W.scales.reshape(-1)])
    data = buffer[5:5 + W.data.numel()].view(W.data.shape)
    again = hip.Fp8Weight(data, buffer[5 + W.data.numel():].view(W.scales.shape),
                          K, N)
    for x in (X, X.to(torch.bfloat16)):
        assert torch.equal(hip.fp8_linear(x, again), hip.fp8_linear(x, W))


# --------------------------------------------------------------- transforms
def test_tangents_go_through():
    """Forward mode: a dual tensor asks for no gradient in reverse, and its
    tangent is as on the CPU."""
    g = gen(3)
    T, dT = torch.randn(2, 20, 8, generator=g)
    ids = torch.randint(-1, 21, (6, 5), generator=g)
    w, dw = torch.rand(2, 6, 5, generator=g)
    x, dx = torch.randn(2, 4, 9, generator=g)
    dy, ddy = torch.randn(2, 6, 8, generator=g)

    def tangents(device):
        def dual(a, b):
            return fwd.make_dual(a.to(device), b.to(device))
        i = ids.to(device)
        with fwd.dual_level():
            out = [embed_tokens(dual(T, dT), i, 2.0),
                   sum_tokens(dual(T, dT), i, w.to(device), 0.5),
                   sum_tokens(T.to(device), i, dual(w, dw)),
                   token_table_grad(dual(dy, ddy), i, 20, w.to(device)),
                   token_table_grad(dy.to(device), i, 20, dual(w, dw)),
                   dropout(dual(x, dx), 0.3, 5, 1)]
            out = [fwd.unpack_dual(y).tangent for y in out]
            assert all(t is not None for t in out)
            return [t.cpu() for t in out]

    # sums of up to ten terms under 20: ten roundings of 2^-24 a side
    for a, b in zip(tangents("cpu"), tangents("cuda")):
        assert torch.allclose(a, b, atol=4e-5)


def test_sparse_scores_do_not_lose_a_tangent():
    """torch has no forward mode for CSR rows, and says so."""
    X = torch.eye(6).to_sparse_csr().cuda()
    W = torch.ones(6, 2, device="cuda")
    with fwd.dual_level():
        with pytest.raises(NotImplementedError):
            csr_matmul(X, fwd.make_dual(W, W))


def test_function_transforms():
    """vmap and jvp hand over tensors without memory of their own."""
    g = gen(4)
    x = torch.randn(3, 40, generator=g).cuda()
    got = torch.func.vmap(lambda a: dropout(a, 0.4, 7, 2))(x)
    want = torch.stack([dropout(a, 0.4, 7, 2) for a in x])
    assert torch.allclose(got, want)
    _, t = torch.func.jvp(lambda a: dropout(a, 0.4, 7, 2), (x,), (x,))
    assert torch.allclose(t, dropout(x, 0.4, 7, 2))


# ------------------------------------------------------------ types, shapes
def test_types_that_the_cpu_takes():
    g = gen(5)
    T = torch.randn(30, 12, generator=g)
    ids = torch.randint(-1, 31, (8, 6), generator=g)
    w = torch.rand(8, 6, generator=g)
    dy = torch.randn(8, 12, generator=g)
    for t in TYPES:
        for wt in (torch.float64, torch.float32, torch.bfloat16, torch.float16):
            for it in (torch.int64, torch.int32, torch.int16, torch.int8):
                outs = []
                for dev in ("cpu", "cuda"):
                    a, i, v, d = (T.to(t).to(dev), ids.to(it).to(dev),
                                  w.to(wt).to(dev), dy.to(t).to(dev))
                    outs.append((embed_tokens(a, i, 1.5), sum_tokens(a, i, v, 0.5),
                                 token_table_grad(d, i, 30, v, 0.5),
                                 token_table_grad(d, i, 30, v, 0.5,
                                                  out=a.clone().float())))
                for a, b in zip(*outs):
                    assert a.dtype == b.dtype
                    # both sides sum in 32 bits and round once; sums of ten
                    # and fewer terms, whose roundings may fall either way
                    step = torch.finfo(a.dtype).eps
                    assert torch.allclose(a.float(), b.cpu().float(),
                                          rtol=step, atol=1e-5), (t, wt, it)


def test_gradient_of_a_single_lookup(hip):
    """Ids of no dimension, and rows of no columns."""
    T = torch.randn(5, 3, device="cuda")
    one = torch.tensor(2, device="cuda")
    y = hip.embedding_lookup(T, one)
    assert torch.equal(y, T[2])
    d = hip.embedding_grad(y, hip.embedding_plan(one, 5))
    want = torch.zeros(5, 3, device="cuda")
    want[2] = T[2]
    assert torch.equal(d, want)
    ids = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    y = hip.embedding_lookup(T[:, :0], ids)
    assert y.shape == (2, 4, 0)
    assert hip.embedding_grad(y, hip.embedding_plan(ids, 5)).shape == (5, 0)


def test_a_plan_used_on_another_stream_keeps_its_memory(hip):
    g = gen(9)
    ids, dy = some_ids(40000, 900, g), torch.randn(40000, 16, generator=g).cuda()
    plan = hip.embedding_plan(ids, 900)
    want = hip.embedding_grad(dy, plan)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        torch.cuda._sleep(10 ** 8)
        got = hip.embedding_grad(dy, plan)
    plan.record_stream(other)
    dy.record_stream(other)
    at, size = plan.keys.data_ptr(), plan._kept.numel()
    del plan
    # what is freed on this stream would be handed out again at once
    others = [torch.empty(size, dtype=torch.int32, device="cuda")
              for _ in range(3)]
    assert all(t.data_ptr() != at for t in others)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("share,sparse", [(0.03, True), (0.3, False)])
@pytest.mark.parametrize("intercept", [False, True])
def test_filled_rows_with_an_intercept_are_fitted_dense(monkeypatch, share,
                                                        sparse, intercept):
    """As before there were kernels for CSR rows, which many stored entries make
    slower; without an intercept those take the place of the library's."""
    calls, t_matmul = [], SparseRows.t_matmul
    monkeypatch.setattr(SparseRows, "t_matmul", lambda self, D:
                        calls.append(1) or t_matmul(self, D))
    g = gen(10)
    X = torch.randn(300, 200, generator=g) * (
        torch.rand(300, 200, generator=g) < share)
    y = torch.randint(0, 3, (300,), generator=g).cuda()
    fits = [cls(LeastSquaresGradient(), 1, 1e-3, fit_intercept=intercept).fit(
        ka.from_rows(A), ka.from_rows(y))
        for cls, A in ((DenseLBFGSwithL2, X.cuda()),
                       (SparseLBFGSwithL2, X.to_sparse_csr().cuda()))]
    assert bool(calls) == (sparse or not intercept)
    assert torch.allclose(fits[0].W, fits[1].W, rtol=1e-4, atol=1e-6)


def test_weights_of_bags_have_the_ids_shape(hip):
    """Weights of another shape with as many elements would go to other ids."""
    g = gen(11)
    T, dy = torch.randn(9, 3, generator=g), torch.randn(4, 3, generator=g)
    ids, w = torch.randint(-1, 9, (4, 6), generator=g), torch.rand(4, 6, generator=g)
    for v in (w[:, :1], w[0], w[:1, :1], w):
        # six roundings of sums of six terms under 4, a side
        assert torch.allclose(sum_tokens(T.cuda(), ids.cuda(), v.cuda()).cpu(),
                              sum_tokens(T, ids, v), atol=12 * 2 ** -24 * 24)
        assert torch.allclose(
            token_table_grad(dy.cuda(), ids.cuda(), 9, v.cuda()).cpu(),
            token_table_grad(dy, ids, 9, v), atol=48 * 2 ** -24 * 96)
    for v in (w.t(), w.reshape(-1), w[None]):
        with pytest.raises((ValueError, RuntimeError)):
            sum_tokens(T.cuda(), ids.cuda(), v.cuda())
        with pytest.raises((ValueError, RuntimeError)):
            token_table_grad(dy.cuda(), ids.cuda(), 9, v.cuda())
    for v in (w.t(), w[None]):
        with pytest.raises(ValueError, match="weights"):
            hip.embedding_bag(T.cuda(), ids.cuda(), weights=v.cuda())
    assert torch.equal(
        hip.embedding_bag(T.cuda(), ids.cuda(), weights=w.reshape(-1).cuda()),
        hip.embedding_bag(T.cuda(), ids.cuda(), weights=w.cuda()))


def test_sums_do_not_land_on_what_is_still_read(hip):
    flat = torch.ones(64, device="cuda")
    ids = torch.arange(8, device="cuda") % 4
    dy, plan = torch.ones(8, 3, device="cuda"), hip.embedding_plan(ids, 4)
    out = flat[4:16].view(4, 3)
    for w in (flat[:8], flat[15:23], flat[6:14]):
        with pytest.raises(ValueError, match="weights"):
            hip.embedding_grad(dy, plan, w, out=out, accumulate=True)
    hip.embedding_grad(dy, plan, flat[16:24], out=out, accumulate=True)
    torch.cuda.synchronize()
    assert out.eq(3).all() and flat[:4].eq(1).all() and flat[16:].eq(1).all()


def captured(step):
    """A graph of `step` and what it returned while it was recorded."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,K,N", [(200, 4100, 130), (300, 5000, 1000),
                                   (4300, 520, 1100), (1025, 8321, 2050)])
def test_large_products_in_a_graph(hip, dtype, M, K, N):
    """Their workspace lies in the graph's own memory: replays between eager
    calls of the same sizes."""
    g = gen(M)
    X = torch.randn(M, K, generator=g).to(dtype).cuda()
    W = hip.fp8_pack(torch.randn(K, N, generator=g).cuda())
    graph, y = captured(lambda: hip.fp8_linear(X, W))
    for _ in range(3):
        X.mul_(-1.5)
        want = hip.fp8_linear(X, W)
        graph.replay()
        other = hip.fp8_linear(X, W)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(other, want)


def test_two_graphs_of_sums_that_share_memory(hip):
    """Long bags, their join, a sort by digits and an update in place, recorded
    twice into one pool and replayed in turn."""
    g = gen(12)
    V, D, n = 30000, 33, 20000
    T, dy = torch.randn(V, D, generator=g).cuda(), torch.randn(4, D, generator=g).cuda()
    ids = [some_ids(n, V, g) for _ in range(2)]
    offsets = some_offsets([9000, 0, 10990, 10])
    w = torch.rand(n, generator=g).cuda()

    def step(k, table):
        y = hip.embedding_bag(table, ids[k], offsets, w)
        plan = hip.embedding_plan(ids[k], V, offsets)
        hip.embedding_grad(dy, plan, w, -0.01, out=table, accumulate=True)
        return y

    eager = T.clone()
    step(0, T.clone())
    pool, graphs, outs = torch.cuda.graph_pool_handle(), [], []
    for k in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[k], pool=pool):
            outs.append(step(k, T))
    for k in (0, 1, 1, 0, 1):
        graphs[k].replay()
        got = outs[k].clone()
        want = step(k, eager)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(T, eager)


def test_negated_views(hip):
    """The imaginary part of a conjugate is a view whose sign torch puts off:
    its memory holds the opposite."""
    g = gen(13)

    def negated(*shape):
        z = torch.randn(*shape, 2, generator=g).cuda()
        n = torch.view_as_complex(z).conj().imag
        assert n.is_neg() and torch.equal(n, -z[..., 1])
        return n

    ids = some_ids(60, 9, g)
    plan = hip.embedding_plan(ids, 9)
    X, W, b = negated(7, 200), negated(200, 5), negated(5)
    for D in (1, 6):
        for T in (negated(9, D), torch._neg_view(torch.randn(9, D, generator=g).cuda())):
            real = T.clone()
            assert not real.is_neg()
            for f in (lambda t: hip.embedding_lookup(t, ids),
                      lambda t: hip.embedding_bag(t, ids.view(6, 10)),
                      lambda t: hip.dropout(t, 0.3, 1, 2),
                      lambda t: hip.sym_rectify(t),
                      lambda t: hip.fp8_pack(t).dequantise()):
                assert torch.equal(f(T), f(real))
    for dy in (negated(60, 3), negated(60, 1)):
        w = negated(60)
        assert torch.equal(hip.embedding_grad(dy, plan, w),
                           hip.embedding_grad(dy.clone(), plan, w.clone()))
    packed = hip.fp8_pack(W)
    assert torch.equal(hip.fp8_linear(X, packed, b),
                       hip.fp8_linear(X.clone(), hip.fp8_pack(W.clone()), b.clone()))
    one = negated(7, 1)
    thin = hip.fp8_pack(torch.ones(1, 3, device="cuda"))
    assert torch.equal(hip.fp8_linear(one, thin), hip.fp8_linear(one.clone(), thin))
    out = torch._neg_view(torch.ones(9, 3, device="cuda"))
    with pytest.raises(RuntimeError, match="negated"):
        hip.embedding_grad(torch.ones(60, 3, device="cuda"), plan, out=out)
    with pytest.raises(RuntimeError, match="negated"):
        hip.dropout(torch.ones(9, 3, device="cuda"), 0.5, 1, out=out)


def test_tensors_without_memory_are_refused(hip):
    """Fake tensors and zeros that torch has not made have no address: nothing
    is launched for them, not for one of several arguments either."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    real = dict(T=torch.ones(6, 8, device="cuda"), w=torch.ones(5, device="cuda"),
                ids=torch.arange(5, device="cuda"),
                off=torch.tensor([0, 2, 5], device="cuda"),
                dy=torch.ones(2, 8, device="cuda"), b=torch.ones(3, device="cuda"),
                step=torch.ones(1, dtype=torch.int64, device="cuda"),
                X=torch.ones(4, 6, device="cuda"), W=torch.ones(6, 3, device="cuda"))
    plan = hip.embedding_plan(real["ids"], 6, real["off"])
    packed = hip.fp8_pack(real["W"])
    calls = {
        ("T", "ids"): lambda T, ids, **k: hip.embedding_lookup(T, ids),
        ("T", "ids", "off", "w"): lambda T, ids, off, w, **k:
            hip.embedding_bag(T, ids, off, w),
        ("ids", "off"): lambda ids, off, **k: hip.embedding_plan(ids, 6, off),
        ("dy", "w"): lambda dy, w, **k: hip.embedding_grad(dy, plan, w),
        ("X", "step"): lambda X, step, **k: hip.dropout(X, 0.5, 1, step),
        ("W",): lambda W, **k: hip.fp8_pack(W),
        ("X", "b"): lambda X, b, **k: hip.fp8_linear(X, packed, b),
    }
    for names, call in calls.items():
        call(**real)
        for name in names:
            # zeros of a call that copies its argument are made by the copy
            zero = torch._efficientzerotensor(
                real[name].shape, dtype=real[name].dtype, device="cuda")
            try:
                got = call(**{**real, name: zero})
            except RuntimeError as e:
                assert "memory" in str(e), e
            else:
                want = call(**{**real, name: zero.clone()})
                if isinstance(want, torch.Tensor):
                    assert torch.equal(got, want)
                else:
                    assert all(torch.equal(u, v) for u, v in zip(
                        vars(got).values(), vars(want).values())
                        if isinstance(u, torch.Tensor))
            with FakeTensorMode():
                fake = torch.empty(real[name].shape, dtype=real[name].dtype,
                                   device="cuda")
            with pytest.raises(RuntimeError, match="memory"):
                call(**{**real, name: fake})
        # a mode that makes every result a fake one takes no real argument
        with FakeTensorMode():
            with pytest.raises((RuntimeError, AssertionError)):
                call(**real)
    torch.cuda.synchronize()


# -------------------------------------------------------------- large sizes
def test_more_ids_than_a_launch_takes(hip):
    """2^32 threads of a launch are 2^34 rows of one column."""
    n = 2 ** 34 + 37
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    T = torch.tensor([[1.0], [2.0], [3.0]], device="cuda").to(torch.bfloat16)
    at = torch.tensor([0, 2 ** 31, 2 ** 33 - 1, 2 ** 33, 2 ** 33 + 1, 2 ** 34 - 1,
                       2 ** 34, 2 ** 34 + 36], device="cuda")
    ids[at] = torch.tensor([2, 1, 2, 1, -1, 2, 1, 2], dtype=torch.int32,
                           device="cuda")
    got = hip.embedding_lookup(T, ids)
    assert got[at, 0].tolist() == [3, 2, 3, 2, 0, 3, 2, 3]
    for p in at[1:].tolist():
        near = got[p - 200:p + 36, 0]
        assert near.eq(1).sum() >= near.numel() - 4 and near.ne(0).sum() >= \
            near.numel() - 1
    del ids, got, near
    torch.cuda.empty_cache()


def test_more_columns_of_weights_than_a_launch_takes(hip):
    """2^32 threads of a launch are 2^26 chunks of 16 columns, 137 GB."""
    N = 2 ** 30 + 21
    W = torch.randn(1, N, device="cuda", dtype=torch.bfloat16)
    packed = hip.fp8_pack(W)
    got = hip.fp8_linear(torch.ones(2, 1, device="cuda", dtype=torch.bfloat16),
                         packed)
    for a, b in ((0, 100), (2 ** 29 - 50, 2 ** 29 + 50), (2 ** 30 - 50, N)):
        want = hip.fp8_round(W[:, a:b].t().float()).t()
        # one product, whose four bits bfloat16 holds
        assert torch.equal(got[:, a:b].float(), want.expand(2, -1))
    del W, packed, got
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1001, 1024])
@pytest.mark.parametrize("over", [-1, 1])
def test_lookup_at_the_cache_border(hip, dtype, D, over):
    """Just under and just over 32 MB of output, stored through and past the
    caches; an odd D lets neighbouring lanes write the same elements."""
    size = torch.finfo(dtype).bits // 8
    n = (32 << 20) // (D * size) + over
    g = gen(D + over)
    T = torch.randn(3001, D, generator=g).to(dtype).cuda()
    ids = some_ids(n, 3001, g)
    ok = (ids >= 0) & (ids < 3001)
    for scale in (1.0, 2.0):
        want = T[ids.clamp(0, 3000)] * scale
        want[~ok] = 0
        assert torch.equal(hip.embedding_lookup(T, ids, scale), want)


@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("D,over", [(1001, -1), (1001, 1), (512, 1)])
def test_gradient_at_the_cache_border(hip, src, out, D, over):
    """Just under and just over 32 MB of gradients that are read once, onto just
    under and just over 32 MB of sums."""
    n = (32 << 20) // (D * (torch.finfo(src).bits // 8)) + 1 + over
    V = (32 << 20) // (D * (torch.finfo(out).bits // 8)) + over
    g = gen(D + over)
    ids = some_ids(n, V, g, hot=0.05)
    dy = torch.randn(n, D, generator=g).to(src).cuda()
    got = hip.embedding_grad(dy, hip.embedding_plan(ids, V), scale=0.5, dtype=out)
    check(got, *sums64(dy, torch.arange(n), ids, None, V, 0.5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,hot", [(900, 1), (900, 600), (5000, 9), (5000, 600),
                                   (20000, 1), (20000, 5000), (20000, 20000)])
@pytest.mark.parametrize("D", [1, 37, 130])
def test_in_place_step_of_a_large_table(hip, dtype, n, hot, D):
    """Fewer tokens than table rows, one of them `hot` times: rows that do not
    occur keep their bits, those that do are off by their sum's roundings."""
    V, g = 50000, gen(n + hot + D)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[torch.randperm(n, generator=g)[:hot]] = V // 3
    dy = torch.randn(n, D, generator=g).to(dtype).cuda()
    flat = torch.randn(V, D + 9, generator=g).to(dtype).cuda()
    table, before = flat[:, 3:3 + D], flat.clone()
    hip.embedding_grad(dy, hip.embedding_plan(ids.cuda(), V), scale=-0.25,
                       out=table, accumulate=True)
    want, mag, m = sums64(dy, torch.arange(n), ids, None, V, -0.25)
    old = before[:, 3:3 + D].cpu().double()
    seen = torch.zeros(V, dtype=torch.bool)
    seen[ids] = True
    check(table.cpu()[seen], (want + old)[seen], (mag + old.abs())[seen],
          m[seen] + 2)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    a, b = flat.cpu().view(bits), before.cpu().view(bits)
    assert torch.equal(a[~seen], b[~seen])
    assert torch.equal(a[:, :3], b[:, :3]) and torch.equal(a[:, 3 + D:], b[:, 3 + D:])


@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("D", [1, 33, 256])
def test_weighted_bag_gradient(hip, src, D):
    lens = [3, 1000, 0, 0, 130, 2, 4000, 7] + [11] * 300
    n, V, g = sum(lens), 61, gen(D)
    ids, offsets = some_ids(n, V, g), some_offsets(lens)
    w = torch.randn(n, generator=g).cuda()
    dy = torch.randn(len(lens), D, generator=g).to(src).cuda()
    bag = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    for out in TYPES:
        got = hip.embedding_grad(dy, hip.embedding_plan(ids, V, offsets), w, 1.5,
                                 dtype=out)
        check(got, *sums64(dy, bag, ids, w, V, 1.5))


@pytest.mark.parametrize("D", [1024, 1025, 1030])
def test_bags_of_a_table_over_32_bit_places(hip, D):
    """Over 2^31 elements: rows read through 64-bit offsets, in units that a
    row's length allows, or one by one where it allows none."""
    V, g = 2 ** 22 + 3, gen(D)
    rows = torch.tensor([0, 5, V // 2, V - 2, V - 1])
    table = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    table[rows.cuda()] = torch.randn(5, D, generator=g).to(torch.bfloat16).cuda()
    lens = [3, 0, 700, 1, 5000, 40]
    n = sum(lens)
    ids = rows[torch.randint(0, 5, (n,), generator=g)]
    ids[::9] = V
    w = torch.randn(n, generator=g).cuda()
    got = hip.embedding_bag(table, ids.cuda(), some_offsets(lens), w, 0.5)
    few = torch.searchsorted(rows, ids)
    few[ids == V] = -1
    bag = torch.repeat_interleave(torch.arange(6), torch.tensor(lens))
    check(got, *sums64(table[rows.cuda()], few, bag, w, 6, 0.5))
    del table
    torch.cuda.empty_cache()
