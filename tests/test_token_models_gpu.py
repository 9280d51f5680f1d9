"""The embedding, dropout and 8-bit operators as the framework uses them, and
what they refuse."""

import pytest
import torch

import keystone_amd as ka
from keystone_amd import hip
from keystone_amd.ops.learning import (
    DenseLBFGSwithL2, EmbeddingClassifierEstimator, LeastSquaresGradient,
    LinearMapper, LogisticGradient, LogisticRegressionEstimator,
    LogisticRegressionModel, NaiveBayesModel, SparseLBFGSwithL2)
from keystone_amd.ops.learning.sparse_rows import SparseRows, csr_matmul
from keystone_amd.ops.nlp.embedding import (embed_tokens, sum_tokens,
                                            token_table_grad)
from keystone_amd.ops.stats import dropout

pytestmark = pytest.mark.gpu


def sparse(n, d, share, seed=0):
    g = torch.Generator().manual_seed(seed)
    X = torch.randn(n, d, generator=g) * (
        torch.rand(n, d, generator=g) < share)
    X[n // 2] = 0
    return X


def test_sparse_rows_multiply():
    X = sparse(90, 700, 0.05)
    csr = X.to_sparse_csr().cuda()
    g = torch.Generator().manual_seed(1)
    for k in (1, 2, 20, 147):
        for extra in (False, True):
            W = torch.randn(700 + extra, k, generator=g).cuda()
            D = torch.randn(90, k, generator=g).cuda()
            S = SparseRows(csr, extra)
            assert S.shape == (90, 700 + extra)
            A = torch.cat([X, torch.ones(90, extra)], 1).double()
            for got, want, mag in (
                    (S @ W, A @ W.cpu().double(),
                     A.abs() @ W.cpu().double().abs()),
                    (S.t_matmul(D), A.t() @ D.cpu().double(),
                     A.t().abs() @ D.cpu().double().abs())):
                # at most 703 roundings in a sum
                assert ((got.cpu().double() - want).abs()
                        <= 703 * 2.0 ** -24 * mag + 1e-30).all()


def test_sparse_scores_keep_refusals_and_gradients():
    X = sparse(30, 40, 0.2).to_sparse_csr().cuda()
    for k in (39, 41):
        with pytest.raises(RuntimeError):
            csr_matmul(X, torch.randn(k, 3, device="cuda"))
        with pytest.raises(RuntimeError):
            LogisticRegressionModel(torch.randn(k, 3, device="cuda")
                                    ).apply_batch(X)
        with pytest.raises(RuntimeError):
            NaiveBayesModel(torch.zeros(3, device="cuda"),
                            torch.randn(k, 3, device="cuda")).apply_batch(X)
    W = torch.randn(40, 3, device="cuda", requires_grad=True)
    csr_matmul(X, W).sum().backward()
    want = X.to_dense().cpu().double().sum(0)
    assert torch.allclose(W.grad[:, 0].cpu().double(), want, atol=1e-5)
    w = torch.randn(40, device="cuda")
    assert csr_matmul(X, w).shape == (30,)


@pytest.mark.parametrize("grad", [LeastSquaresGradient(), LogisticGradient()])
@pytest.mark.parametrize("intercept", [False, True])
def test_sparse_fit_is_the_dense_fit(grad, intercept):
    """One step of either solver from the same start: the line search's first
    gradient differs by roundings alone."""
    X = sparse(200, 50, 0.2)
    y = torch.randint(0, 3, (200,), generator=torch.Generator().manual_seed(2))
    fits = [cls(grad, 1, 1e-3, fit_intercept=intercept).fit(
        ka.from_rows(A), ka.from_rows(y.cuda()))
        for cls, A in ((DenseLBFGSwithL2, X.cuda()),
                       (SparseLBFGSwithL2, X.to_sparse_csr().cuda()))]
    assert torch.allclose(fits[0].W, fits[1].W, rtol=1e-4, atol=1e-6)
    if intercept:
        assert torch.allclose(fits[0].b, fits[1].b, rtol=1e-4, atol=1e-6)


def test_a_users_gradient_still_gets_the_tensor():
    seen = []

    class Own(LeastSquaresGradient):
        def compute(self, W, X, Y):
            seen.append(X)
            return super().compute(W, X, Y)

    X = sparse(40, 12, 0.3).to_sparse_csr().cuda()
    SparseLBFGSwithL2(Own(), 2).fit(ka.from_rows(X),
                                    ka.from_rows(torch.randn(40, 2).cuda()))
    assert seen and all(isinstance(x, torch.Tensor) for x in seen)


def test_text_models_score_sparse_rows():
    X = sparse(64, 300, 0.1).abs()
    csr = X.to_sparse_csr().cuda()
    W, p = torch.randn(300, 20).cuda(), torch.randn(20).cuda()
    got = NaiveBayesModel(p, W).apply_batch(csr)
    want = NaiveBayesModel(p, W).apply_batch(X.cuda())
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-4)
    got = LogisticRegressionModel(W, p, True).apply_batch(csr)
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-4)
    y = torch.arange(64).cuda() % 2
    model = LogisticRegressionEstimator(2, num_iters=3).fit(
        ka.from_rows(csr), ka.from_rows(y))
    assert model.apply_batch(csr).shape == (64,)


def test_classifier_gradients_match_the_cpu():
    """The same batch, the same mask.  Sums of at most 40 terms, a chain of
    four products: 1e-5 of the largest gradient covers the roundings."""
    g = torch.Generator().manual_seed(3)
    est = EmbeddingClassifierEstimator(500, 7, dim=33, dropout=0.25, seed=1)
    ids = torch.randint(-1, 501, (64, 40), generator=g)
    y = torch.randint(0, 7, (64,), generator=g)
    host = est.gradients(est.initial("cpu"), ids, y, 64, 9, 4)
    card = est.gradients(est.initial("cuda"), ids.cuda(), y.cuda(), 64, 9, 4)
    for a, b in zip([host[0], *host[1]], [card[0], *card[1]]):
        assert (a - b.cpu()).abs().max() <= 1e-5 * a.abs().max()


def test_train_then_serve_in_8_bits_from_a_graph():
    """The run that the operators make together: lookup and its gradient,
    dropout, then a served model with 8-bit class weights, captured."""
    from keystone_amd.workflow.capture import capture_apply
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(-1, 900, (300, 24), generator=g).cuda()
    y = torch.randint(0, 147, (300,), generator=g).cuda()
    est = EmbeddingClassifierEstimator(900, 147, dim=256, num_epochs=2,
                                       batch_size=64, dropout=0.2)
    model = est.fit(ka.from_rows(ids), ka.from_rows(y))
    again = est.fit(ka.from_rows(ids), ka.from_rows(y))
    assert torch.equal(model.table, again.table)      # no atomics: same bits
    served = model.quantize()
    want = served.apply_batch(ids)
    h = model.apply_batch(ids)
    assert want.shape == h.shape == (300, 147)
    fast = capture_apply(ka.Identity().and_then(served), ids[:64])
    for k in range(4):
        batch = ids[k * 32:k * 32 + 64]
        got = fast.apply_batch(batch)
        torch.cuda.synchronize()
        assert torch.equal(got, served.apply_batch(batch))


def test_training_step_in_a_graph_with_a_moving_step():
    """Lookup, dropout, gradient and update as one graph: a replay is the
    eager step with the next dropout."""
    g = torch.Generator().manual_seed(5)
    V, D = 400, 64
    T = torch.randn(V, D, generator=g).cuda()
    ids = torch.randint(-1, V, (1000,), generator=g).cuda()
    dy = torch.randn(1000, D, generator=g).cuda()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def one(T, at):
        y = hip.dropout(hip.embedding_lookup(T, ids, 8.0), 0.1, 3, at)
        d = hip.dropout(dy, 0.1, 3, at)
        hip.embedding_grad(d, hip.embedding_plan(ids, V), scale=-0.1, out=T,
                           accumulate=True)
        return y

    own = T.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        one(T.clone(), step)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = one(T, step)
        step.add_(1)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = one(own, k)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(T, own)


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(6)
    T = torch.randn(3000, 128, generator=g).cuda()
    X, W = torch.randn(64, 2048, generator=g).cuda(), hip.fp8_pack(
        torch.randn(2048, 100, generator=g).cuda())
    ids = [torch.randint(0, 3000, (40, 500), generator=g).cuda()
           for _ in range(2)]
    want = [(hip.embedding_bag(T, i), hip.fp8_linear(X * (k + 1), W),
             hip.embedding_plan(i, 3000).order)
            for k, i in enumerate(ids)]
    streams = [torch.cuda.Stream() for _ in ids]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for k, (s, i) in enumerate(zip(streams, ids)):
            with torch.cuda.stream(s):
                got.append((hip.embedding_bag(T, i),
                            hip.fp8_linear(X * (k + 1), W),
                            hip.embedding_plan(i, 3000).order))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want)
                   for a, b in zip(x, y))


def test_refusals():
    T = torch.ones(6, 4, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    off = torch.tensor([0, 3], device="cuda")
    plan = hip.embedding_plan(ids, 6)
    dy = torch.ones(3, 4, device="cuda")
    W = hip.fp8_pack(T)
    w = torch.ones(3, device="cuda")
    refused = [
        (RuntimeError, lambda: hip.embedding_lookup(T.double(), ids)),
        (RuntimeError, lambda: hip.embedding_lookup(T, ids.float())),
        (RuntimeError, lambda: hip.embedding_lookup(T, ids.cpu())),
        (ValueError, lambda: hip.embedding_lookup(T[0], ids)),
        (ValueError, lambda: hip.embedding_bag(T, ids)),
        (ValueError, lambda: hip.embedding_bag(T, ids[None], off)),
        (ValueError, lambda: hip.embedding_bag(T, ids, off[:0])),
        (RuntimeError, lambda: hip.embedding_bag(T, ids, off.float())),
        (ValueError, lambda: hip.embedding_bag(T, ids, off, w[:2])),
        (RuntimeError, lambda: hip.embedding_bag(T, ids, off, w.double())),
        (RuntimeError, lambda: hip.embedding_bag(T, ids, off, w.cpu())),
        (ValueError, lambda: hip.embedding_plan(ids, -1)),
        (ValueError, lambda: hip.embedding_plan(ids, 2 ** 29 + 1)),
        (ValueError, lambda: hip.embedding_bag(
            T, ids[:0, None].expand(0, 3).new_empty(2 ** 29 + 1, 0))),
        (ValueError, lambda: hip.embedding_plan(ids, 6, pooled=True)),
        (ValueError, lambda: hip.embedding_grad(dy[:2], plan)),
        (RuntimeError, lambda: hip.embedding_grad(dy.double(), plan)),
        (RuntimeError, lambda: hip.embedding_grad(dy, plan,
                                                  dtype=torch.float64)),
        (ValueError, lambda: hip.embedding_grad(dy, plan, accumulate=True)),
        (ValueError, lambda: hip.embedding_grad(dy, plan, out=T[:5])),
        (RuntimeError, lambda: hip.embedding_grad(dy, plan, out=T.double())),
        (RuntimeError, lambda: hip.embedding_grad(
            dy, plan, out=torch.ones(4, 6, device="cuda").t())),
        (RuntimeError, lambda: hip.embedding_grad(dy, plan,
                                                  out=T[:1].expand(6, 4))),
        (ValueError, lambda: hip.embedding_grad(T[:3], plan, out=T)),
        (ValueError, lambda: hip.embedding_grad(dy, plan, w[:1])),
        (RuntimeError, lambda: hip.dropout(T.double(), 0.5, 0)),
        (ValueError, lambda: hip.dropout(T, 1.0, 0)),
        (ValueError, lambda: hip.dropout(T, 0.5, -1)),
        (ValueError, lambda: hip.dropout(T, 0.5, 0, 2 ** 64)),
        (RuntimeError, lambda: hip.dropout(T, 0.5, 0, ids)),
        (RuntimeError, lambda: hip.dropout(T, 0.5, 0, off[:1].int())),
        (RuntimeError, lambda: hip.dropout(T, 0.5, 0, out=T.t())),
        (ValueError, lambda: hip.dropout(T[:5], 0.5, 0, out=T[1:])),
        (RuntimeError, lambda: hip.fp8_pack(T.double())),
        (ValueError, lambda: hip.fp8_pack(T[None])),
        (ValueError, lambda: hip.Fp8Weight(W.data, W.scales, 6, 17)),
        (ValueError, lambda: hip.Fp8Weight(W.data, W.scales, 129, 4)),
        (ValueError, lambda: hip.Fp8Weight(W.data.int(), W.scales, 6, 4)),
        (ValueError, lambda: hip.fp8_linear(T, W)),
        (RuntimeError, lambda: hip.fp8_linear(T[:, :1].double(), W)),
        (RuntimeError, lambda: hip.fp8_linear(
            torch.ones(2, 6, device="cuda"), W.to("cpu"))),
        (ValueError, lambda: hip.fp8_linear(torch.ones(2, 6, device="cuda"),
                                            W, w)),
        (RuntimeError, lambda: hip.fp8_linear(
            torch.ones(2, 6, device="cuda"), W,
            torch.ones(4, device="cuda").double())),
    ]
    for k, (kind, call) in enumerate(refused):
        with pytest.raises(kind):
            call()
            print("not refused:", k)
    torch.cuda.synchronize()


def test_autograd_through_the_operators_is_not_lost():
    """Sums of up to ten terms of at most 20: ten roundings of 2^-24 a side."""
    g = torch.Generator().manual_seed(4)
    table = torch.randn(20, 8, generator=g).cuda()
    ids = torch.randint(-1, 21, (6, 5), generator=g).cuda()
    w = torch.rand(6, 5, generator=g).cuda()
    dy = torch.randn(6, 8, generator=g).cuda()
    t, v = table.clone().requires_grad_(), w.clone().requires_grad_()
    y = dropout(sum_tokens(t, ids, v, 0.5), 0.3, 11, 2)
    y.backward(dy)
    assert torch.allclose(y, dropout(sum_tokens(table, ids, w, 0.5), 0.3, 11, 2),
                          atol=4e-5)
    dh = dropout(dy, 0.3, 11, 2)
    assert torch.allclose(t.grad, token_table_grad(dh, ids, 20, w, 0.5),
                          atol=4e-5)
    want = 0.5 * (embed_tokens(table, ids) * dh.unsqueeze(1)).sum(-1)
    assert torch.allclose(v.grad, want, atol=4e-5)
    with torch.no_grad():
        assert torch.equal(sum_tokens(t, ids, v, 0.5),
                           hip.embedding_bag(table, ids, None, w, 0.5))
