"""Embeddings, dropout and 8-bit linear maps on the CPU: the operators' plain
paths, their refusals, the estimators that use them."""

import numpy as np
import pytest
import torch

import keystone_amd as ka
from keystone_amd import hip
from keystone_amd.models import (NewsgroupsEmbeddingConfig, TimitConfig,
                                 build_newsgroups_embedding, build_timit)
from keystone_amd.ops.learning import (
    BlockLeastSquaresEstimator, BlockLinearMapper,
    EmbeddingClassifierEstimator, LeastSquaresGradient, LinearMapEstimator,
    LinearMapper, LogisticGradient, MiniBatchSGDwithL2, QuantizedEstimator,
    QuantizedLinearMapper)
from keystone_amd.ops.learning.sparse_rows import SparseRows
from keystone_amd.ops.nlp import MeanEmbedding, PadTokens, TokenEmbedding
from keystone_amd.ops.nlp.embedding import (embed_tokens, mean_weights,
                                            sum_tokens, token_table_grad)
from keystone_amd.ops.stats import dropout
from keystone_amd.ops.util import VectorSplitter
from tests.dist_util import run_distributed
from tests.philox import expected, philox


# ------------------------------------------------------------------ dropout
def test_philox_known_answers():
    """The published vectors of the generator."""
    cases = [((0, 0, 0, 0), (0, 0),
              (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
             ((0xffffffff,) * 4, (0xffffffff,) * 2,
              (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
             ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344),
              (0xa4093822, 0x299f31d0),
              (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]
    for c, k, want in cases:
        got = philox(np.array([c], dtype=np.uint32), k)[0]
        assert tuple(int(x) for x in got) == want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16,
                                   torch.float16])
@pytest.mark.parametrize("shape", [(1,), (7,), (33, 65), (0, 3)])
def test_dropout_matches_the_generator(dtype, shape):
    x = torch.randn(shape).to(dtype)
    for p, seed, step in ((0.0, 0, 0), (0.3, 2 ** 64 - 1, 2 ** 64 - 1),
                          (0.9, 5, 2 ** 33)):
        want, _ = expected(x, p, seed, step)
        assert torch.equal(dropout(x, p, seed, step), want)


def test_dropout_refusals():
    x = torch.ones(4)
    for p in (-0.1, 1.0, 2.0, float("nan"), 1 - 2.0 ** -18):
        with pytest.raises(ValueError, match="chance"):
            dropout(x, p, 0)
    for seed, step in ((-1, 0), (0, -1), (2 ** 64, 0), (0, 2 ** 64)):
        with pytest.raises(ValueError, match="2\\^64"):
            dropout(x, 0.5, seed, step)


@pytest.mark.parametrize("grad", [LeastSquaresGradient(), LogisticGradient()])
def test_minibatch_sgd_with_dropout(grad):
    """Against the loop written out; a chance of 0 changes nothing."""
    X, y = torch.randn(60, 9), torch.randint(0, 3, (60,))
    Y = torch.nn.functional.one_hot(y).float()
    for p in (0.0, 0.4):
        got = MiniBatchSGDwithL2(grad, 5, 0.1, 0.25, 1e-3, seed=3, dropout=p
                                 ).fit(ka.from_rows(X), ka.from_rows(y)).W
        W, g = torch.zeros(9, 3), torch.Generator().manual_seed(3)
        for it in range(5):
            idx = torch.randperm(60, generator=g)[:15]
            Xb = dropout(X[idx], p, 3, it) if p else X[idx]
            _, d = grad.compute(W, Xb, Y[idx])
            W = W - 0.1 / (1 + it) ** 0.5 * (d / 15 + 1e-3 * W)
        # the same operations but for the mean, taken in 64 bits there
        assert torch.allclose(got, W, rtol=1e-5, atol=1e-6)


# --------------------------------------------------------------- embeddings
def test_embeddings_by_hand():
    T = torch.tensor([[1., 2], [10, 20], [100, 200]])
    ids = torch.tensor([[0, 2, -1], [-1, 3, -1], [1, 1, 0]])
    assert torch.equal(embed_tokens(T, ids, 2.0)[0],
                       torch.tensor([[2., 4], [200, 400], [0, 0]]))
    w = mean_weights(ids, 3)
    got = sum_tokens(T, ids, w)
    assert torch.allclose(got, torch.tensor([[50.5, 101], [0, 0], [7, 14]]))
    dy = torch.tensor([[2., 4], [1, 1], [3, 6]])
    want = torch.tensor([[2., 4], [2, 4], [1, 2]])
    assert torch.allclose(token_table_grad(dy, ids, 3, w), want)
    out = torch.ones(3, 2)
    assert token_table_grad(dy, ids, 3, w, -1.0, out=out) is out
    assert torch.allclose(out, 1 - want)
    assert torch.equal(MeanEmbedding(T).apply_batch(ids), got)
    assert TokenEmbedding(T, 3.0).apply_batch(ids).shape == (3, 3, 2)


def test_table_gradient_agrees_with_autograd():
    g = torch.Generator().manual_seed(0)
    T = torch.randn(11, 5, generator=g, dtype=torch.float64)
    ids = torch.randint(-1, 12, (7, 6), generator=g)
    w = torch.rand(7, 6, generator=g)
    dy = torch.randn(7, 5, generator=g, dtype=torch.float64)
    T.requires_grad_()
    rows = torch.nn.functional.pad(T, (0, 0, 0, 1))[
        torch.where((ids >= 0) & (ids < 11), ids, 11)]
    ((rows * w.unsqueeze(-1).double()).sum(1) * 0.5 * dy).sum().backward()
    got = token_table_grad(dy, ids, 11, w, 0.5)
    assert torch.allclose(got, T.grad, rtol=1e-12, atol=1e-12)


def test_pad_tokens():
    pad = PadTokens(3)
    ds = pad.apply_dataset(ka.from_items([[5, 6, 7, 8], [1], []]))
    assert ds.data.tolist() == [[5, 6, 7], [1, -1, -1], [-1, -1, -1]]
    assert pad.apply_dataset(ka.from_items([])).data.shape == (0, 3)
    with pytest.raises(ValueError, match="length"):
        PadTokens(0)


def test_embedding_transformers_save_and_load(tmp_path):
    T, ids = torch.randn(6, 4), torch.tensor([[0, 5, -1], [2, 2, 9]])
    for t in (TokenEmbedding(T, 2.0), MeanEmbedding(T, 0.5)):
        pipe = ka.Identity().and_then(t)
        pipe.save(str(tmp_path / type(t).__name__))
        again = ka.Pipeline.load(str(tmp_path / type(t).__name__))
        ds = ka.from_rows(ids)
        assert torch.equal(pipe.apply(ds).get().data,
                           again.apply(ds).get().data)
    for bad in (torch.ones(3), torch.ones(3, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="table"):
            TokenEmbedding(bad)


# ------------------------------------------------------ embedding classifier
def test_classifier_gradients_agree_with_differences():
    """Central differences in 64 bits: the third derivative's term h^2 and
    the roundings 2^-52 / h are both far under 1e-7 at h = 1e-5."""
    est = EmbeddingClassifierEstimator(9, 4, dim=5, dropout=0.3, seed=2)
    params = [p.double() for p in est.initial("cpu")]
    ids = torch.tensor([[0, 3, -1, 8], [1, 1, 2, 9], [-1, -1, -1, -1],
                        [7, 0, 0, 3]])
    y = torch.tensor([0, 3, 1, 2])

    def f():
        return est.gradients(params, ids, y, 4, 11, 6)[0].item()

    _, grads = est.gradients(params, ids, y, 4, 11, 6)
    for p, d in zip(params, grads):
        assert p.shape == d.shape
        for i in range(p.numel()):
            at, h, keep = p.view(-1), 1e-5, p.view(-1)[i].item()
            at[i] = keep + h
            up = f()
            at[i] = keep - h
            down = f()
            at[i] = keep
            assert abs((up - down) / (2 * h) - d.reshape(-1)[i].item()) < 1e-7


def test_classifier_step_in_place_is_the_gradient_step():
    est = EmbeddingClassifierEstimator(9, 4, dim=5, dropout=0.3, seed=2)
    ids, y = torch.randint(-1, 10, (8, 6)), torch.randint(0, 4, (8,))
    params = est.initial("cpu")
    E = params[0].clone()
    _, grads = est.gradients(params, ids, y, 8, 1, 2)
    _, again = est.gradients(params, ids, y, 8, 1, 2, -0.5)
    assert again[0] is None
    assert torch.allclose(params[0], E - 0.5 * grads[0], atol=1e-6)
    seen = torch.zeros(9, dtype=torch.bool)
    seen[ids[(ids >= 0) & (ids < 9)]] = True
    assert torch.equal(params[0][~seen], E[~seen])


def test_classifier_refusals():
    est = EmbeddingClassifierEstimator(9, 4)
    ids = torch.zeros(3, 2, dtype=torch.int64)
    for y in (torch.tensor([0, 4, 1]), torch.tensor([0, -1, 1])):
        with pytest.raises(ValueError, match="labels"):
            est.fit(ka.from_rows(ids), ka.from_rows(y))
    with pytest.raises(ValueError, match="ids"):
        est.fit(ka.from_rows(ids), ka.from_rows(torch.tensor([0, 1])))


def test_newsgroups_embedding_trains_serves_saves(tmp_path):
    from keystone_amd.loaders import synthetic_documents
    docs, labels = synthetic_documents(60, num_classes=3, vocab_size=200,
                                       doc_len=20, seed=4)
    fitted = build_newsgroups_embedding(docs, labels, NewsgroupsEmbeddingConfig(
        num_classes=3, num_words=150, doc_len=16, dim=8, num_epochs=2,
        batch_size=25)).fit()
    pred = fitted.apply(docs).get().data
    assert pred.shape == (60,) and int(pred.min()) >= 0 and int(pred.max()) < 3
    fitted.save(str(tmp_path / "m"))
    again = ka.Pipeline.load(str(tmp_path / "m")).apply(docs).get().data
    assert torch.equal(pred, again)


def _fit_classifier(rank, world):
    g = torch.Generator().manual_seed(rank)
    n = 30 if rank == 0 else 17                  # shards of unlike size
    ids = torch.randint(-1, 50, (n, 6), generator=g)
    y = torch.randint(0, 3, (n,), generator=g)
    m = EmbeddingClassifierEstimator(50, 3, dim=7, num_epochs=2, batch_size=8,
                                     dropout=0.2, seed=5).fit(
        ka.from_rows(ids), ka.from_rows(y))
    return [m.table, m.head.W, m.head.b]


def test_classifier_is_the_same_on_all_ranks():
    a, b = run_distributed(_fit_classifier, 2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------- 8-bit linear
def test_fp8_round_by_definition():
    """Against the grid written out: multiples of 2^(exponent - 3), from
    2^-9 of the block's scale on, halves to even."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 300, generator=g) * torch.exp(
        3 * torch.randn(5, 300, generator=g))
    x[2, 128:256] = 0
    x[3, :128] *= 1e-30
    got = hip.fp8_round(x).double()
    for r in range(5):
        for k in range(0, 300, 128):
            b = x[r, k:k + 128].double()
            top = b.abs().max().item()
            e = 0
            if top:
                e = max(-117, int(np.ceil(np.log2(top / 448))))
                assert 448 * 2.0 ** (e - 1) < top <= 448 * 2.0 ** e
            v = (b / 2.0 ** e).numpy()
            power = np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6)))
            unit = 2.0 ** (power - 3)
            want = np.round(v / unit) * unit * 2.0 ** e
            assert np.array_equal(got[r, k:k + 128].numpy(), want)


def test_quantized_mapper_matches_its_rounded_operands(tmp_path):
    W, b = torch.randn(300, 17), torch.randn(17)
    X = torch.randn(9, 300)
    q = LinearMapper(W, b).quantize()
    want = hip.fp8_round(X) @ hip.fp8_round(W.t()).t() + b
    assert torch.allclose(q.apply_batch(X), want, rtol=1e-5, atol=1e-5)
    assert torch.allclose(q.apply(X[0]), want[0], rtol=1e-5, atol=1e-5)
    assert q.apply_batch(X.double()).dtype == torch.float64
    # off by 2^-4 of each factor at most, and a little for the small ones
    exact, mag = X @ W + b, X.abs() @ W.abs()
    assert ((q.apply_batch(X) - exact).abs() <= 0.14 * mag).all()
    ka.Identity().and_then(q).save(str(tmp_path / "q"))
    again = ka.Pipeline.load(str(tmp_path / "q"))
    assert torch.equal(again.apply(ka.from_rows(X)).get().data,
                       q.apply_batch(X))
    with pytest.raises(ValueError, match="features"):
        q.apply_batch(X[:, :299])


def test_quantized_block_mapper_takes_blocks_and_whole_features():
    blocks, b = [torch.randn(64, 5), torch.randn(36, 5)], torch.randn(5)
    m = BlockLinearMapper(blocks, b)
    q, X = m.quantize(), torch.randn(7, 100)
    want = LinearMapper(torch.cat(blocks), b).quantize().apply_batch(X)
    assert torch.equal(q.apply_batch(X), want)
    split = VectorSplitter(64).apply_dataset(ka.from_rows(X))
    assert torch.equal(q.apply_dataset(split).data, want)
    assert torch.equal(q.apply(list(torch.split(X[0], 64))), want[0])
    lazy = BlockLinearMapper(blocks, None, [ka.Identity(), ka.Identity()])
    with pytest.raises(ValueError, match="lazy"):
        lazy.quantize()


def test_quantized_estimator():
    X, Y = torch.randn(50, 12), torch.randn(50, 3)
    ds, ys = ka.from_rows(X), ka.from_rows(Y)
    q = QuantizedEstimator(LinearMapEstimator(0.1)).fit(ds, ys)
    assert isinstance(q, QuantizedLinearMapper)
    want = LinearMapEstimator(0.1).fit(ds, ys).quantize()
    assert torch.equal(q.packed.data, want.packed.data)
    one, two = (QuantizedEstimator(BlockLeastSquaresEstimator(4, 1, lam))
                for lam in (0.1, 0.2))
    assert one.inner_key != two.inner_key
    with pytest.raises(TypeError, match="linear map"):
        QuantizedEstimator(EmbeddingLess()).fit(ds, ys)


class EmbeddingLess(LinearMapEstimator):
    def _fit(self, data, labels):
        return ka.Identity()


def test_timit_with_8_bit_scores():
    from keystone_amd.loaders.synthetic import synthetic_dense
    train, labels = synthetic_dense(200, 40, 5, seed=4, noise=0.5)
    fitted = build_timit(train, labels, TimitConfig(
        input_dim=40, num_features=256, gamma=0.02, num_classes=5,
        block_size=128, num_iter=1, lam=1e-3, fp8_scores=True)).fit()
    assert any(isinstance(t, QuantizedLinearMapper)
               for t in fitted.transformers())
    assert fitted.apply(train).get().data.shape == (200,)


# ----------------------------------------------------------------- refusals
@pytest.mark.skipif(not hip.available(), reason="extension not built")
def test_kernels_refuse_host_tensors():
    T, ids = torch.ones(4, 3), torch.tensor([[0, 1]])
    for call in (lambda: hip.embedding_lookup(T, ids),
                 lambda: hip.embedding_bag(T, ids),
                 lambda: hip.embedding_plan(ids, 4),
                 lambda: hip.dropout(T, 0.5, 0),
                 lambda: hip.fp8_linear(T, hip.fp8_pack(torch.ones(3, 2)))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_sparse_rows_over_the_kernels_sizes_are_left_to_torch(monkeypatch):
    from types import SimpleNamespace
    monkeypatch.setattr(hip, "gpu_ready", lambda: True)

    def rows(n, d, entries, dims=2, grad=False):
        return SimpleNamespace(
            layout=torch.sparse_csr, is_cuda=True, dtype=torch.float32,
            shape=(n, d), dim=lambda: dims, requires_grad=grad,
            values=lambda: SimpleNamespace(numel=lambda: entries))

    most = hip.MAX_TOKENS
    assert SparseRows.supports(rows(most, most, most))
    assert not SparseRows.supports(rows(most + 1, 5, 5))
    assert not SparseRows.supports(rows(5, most + 1, 5))
    assert not SparseRows.supports(rows(5, 5, most + 1))
    assert not SparseRows.supports(rows(5, 5, 5, dims=3))
    assert not SparseRows.supports(rows(5, 5, 5, grad=True))
    with torch.no_grad():
        assert SparseRows.supports(rows(5, 5, 5, grad=True))
