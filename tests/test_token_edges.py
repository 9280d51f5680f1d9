"""The token, dropout and 8-bit operators at their edges, on the CPU."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import keystone_amd as ka
from keystone_amd import hip
from keystone_amd.ops.learning import (EmbeddingClassifierEstimator,
                                       LeastSquaresGradient, LinearMapper,
                                       MiniBatchSGDwithL2)
from keystone_amd.ops.nlp import MeanEmbedding
from keystone_amd.ops.nlp.embedding import sum_tokens, token_table_grad
from keystone_amd.utils.derivatives import differentiated
from tests.dist_util import run_distributed


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


def test_absent_words_weigh_nothing():
    """A word outside the table is no term of a sum whatever its weight, and
    has no gradient."""
    T = torch.randn(4, 3, requires_grad=True)
    ids = torch.tensor([[0, -1, 3], [4, -1, -1]])
    for bad in (float("nan"), float("inf")):
        w = torch.tensor([[2.0, bad, 1.0], [bad, bad, bad]], requires_grad=True)
        y = sum_tokens(T, ids, w)
        assert torch.equal(y[0], 2 * T[0] + T[3]) and y[1].eq(0).all()
        dT, dw = torch.autograd.grad(y.sum(), (T, w))
        want = torch.zeros(4, 3)
        want[0], want[3] = 2, 1
        assert torch.equal(dT, want) and dw[1].eq(0).all() and dw[0, 1] == 0
        assert torch.equal(token_table_grad(torch.ones(2, 3), ids, 4, w.detach()),
                           want)
        # the sum's gradient is linear in the rows' one: its own derivative
        dy = torch.ones(2, 3, requires_grad=True)
        d, = torch.autograd.grad(token_table_grad(dy, ids, 4, w.detach()).sum(), dy)
        assert d[0].eq(3).all() and d[1].eq(0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sums_of_16_bit_tables_round_once(dtype):
    """32 terms of 1 + eps: in 32 bits each partial sum is exact (24 bits, with
    a weight that bfloat16 cannot hold), and the result rounds once."""
    one, weight = 1 + torch.finfo(dtype).eps, 1 + 2.0 ** -8
    T = torch.tensor([[one], [0.25]], dtype=dtype)
    ids = torch.zeros(2, 32, dtype=torch.int64)
    ids[1, 16:] = 1
    w = torch.full((2, 32), weight)
    exact = torch.tensor([[32 * one], [16 * one + 4]], dtype=torch.float64)
    assert torch.equal(sum_tokens(T, ids), exact.to(dtype))
    assert torch.equal(sum_tokens(T, ids, w, 2.0), (exact * 2 * weight).to(dtype))
    dy = torch.tensor([[one], [0.25]], dtype=dtype)
    want = torch.tensor([[32 * one + 4], [4.0]], dtype=torch.float64)
    got = token_table_grad(dy, ids, 2)
    assert got.dtype == dtype and torch.equal(got, want.to(dtype))
    for out in (torch.ones(2, 1), torch.ones(2, 1, dtype=dtype),
                torch.ones(2, 1, dtype=torch.float64)):
        again = token_table_grad(dy, ids, 2, None, 1.0, out)
        assert again is out and torch.equal(out, (want + 1).to(out.dtype))


def test_any_seed_that_torch_takes():
    """Negative seeds too, which torch's generators count modulo 2^64."""
    ids, y = torch.randint(-1, 9, (20, 4)), torch.randint(0, 3, (20,))
    X = torch.randn(20, 5)
    for p in (0.0, 0.3):
        a, b = (EmbeddingClassifierEstimator(
            9, 3, dim=4, num_epochs=1, batch_size=8, dropout=p, seed=s).fit(
            ka.from_rows(ids), ka.from_rows(y)) for s in (-5, 2 ** 64 - 5))
        assert torch.equal(a.table, b.table) and torch.equal(a.head.W, b.head.W)
        a, b = (MiniBatchSGDwithL2(LeastSquaresGradient(), 3, seed=s, dropout=p
                                   ).fit(ka.from_rows(X), ka.from_rows(y)).W
                for s in (-5, 2 ** 64 - 5))
        assert torch.equal(a, b)


def _fit_refused(rank, world, wrong):
    ids, y = torch.zeros(6, 3, dtype=torch.int64), torch.zeros(6, dtype=torch.int64)
    if rank == 1 and wrong == "label":
        y[4] = 7
    elif rank == 1 and wrong == "rows":
        y = y[:5]
    elif rank == 1:
        ids = ids[:, 0]
    try:
        EmbeddingClassifierEstimator(9, 3, dim=4, num_epochs=1).fit(
            ka.from_rows(ids), ka.from_rows(y))
    except ValueError as e:
        return str(e)
    return "fitted"


@pytest.mark.parametrize("wrong,says", [("label", "labels in"), ("rows", "ids"),
                                        ("ids", "ids")])
def test_what_one_rank_refuses_all_ranks_refuse(wrong, says):
    """Or the others would wait for it in the first reduction."""
    other, own = run_distributed(_fit_refused, 2, (wrong,))
    assert says in own and "rank" in other


@pytest.mark.parametrize("off", [1, 4, 8])
def test_packed_weights_from_views_are_aligned(off):
    """The kernels read them 16 bytes at a time; bytes taken out of a larger
    buffer need not lie so."""
    W = hip.fp8_pack(torch.randn(300, 40))

    def moved(t):
        flat = torch.zeros(t.numel() + 64, dtype=torch.uint8)
        at = flat[(off - flat.data_ptr()) % 16:][:t.numel()].view(t.shape)
        at.copy_(t)
        assert at.data_ptr() % 16 == off
        return at

    again = hip.Fp8Weight(moved(W.data), moved(W.scales), 300, 40)
    for a, b in ((again.data, W.data), (again.scales, W.scales)):
        assert a.data_ptr() % 16 == 0 and torch.equal(a, b)


def test_quantized_scores_of_rows_in_several_dimensions():
    """As LinearMapper and BlockLinearMapper: the last dimension is the
    features'."""
    lin = LinearMapper(torch.randn(70, 5), torch.randn(5))
    q = lin.quantize()
    for shape in ((2, 70, 70), (3, 4, 70), (0, 4, 70), (2, 0, 70), (1, 1, 1, 70)):
        X = torch.randn(shape)
        got = q.apply_batch(X)
        assert got.shape == lin.apply_batch(X).shape
        assert torch.equal(got.reshape(-1, 5), q.apply_batch(X.reshape(-1, 70)))
        ds = ka.from_rows(X)
        assert torch.equal(q.apply_dataset(ds).data, got)
    with pytest.raises(ValueError, match="features"):
        q.apply_batch(torch.randn(2, 70, 71))


def test_weights_have_the_ids_shape_or_are_spread_over_it():
    T, ids = torch.randn(9, 3), torch.randint(0, 9, (4, 6))
    w, dy = torch.rand(4, 6), torch.randn(4, 3)
    for v in (w[:, :1], w[0], w[:1, :1], w):
        full = v.expand(4, 6)
        assert torch.equal(sum_tokens(T, ids, v), sum_tokens(T, ids, full))
        assert torch.equal(token_table_grad(dy, ids, 9, v),
                           token_table_grad(dy, ids, 9, full))
    for v in (w.t(), w[:, :5], w.reshape(-1), w[None]):
        with pytest.raises((ValueError, RuntimeError)):
            sum_tokens(T, ids, v)
        with pytest.raises((ValueError, RuntimeError)):
            token_table_grad(dy, ids, 9, v)


def test_bags_of_ids_are_rows():
    T = torch.randn(9, 3)
    for ids in (torch.tensor([1, 2]), torch.zeros(2, 2, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="ids"):
            sum_tokens(T, ids)
        with pytest.raises(ValueError, match="ids"):
            token_table_grad(torch.ones(2, 3), ids, 9)


def test_means_of_64_bit_tables_are_in_64_bits():
    T = torch.randn(5, 4, dtype=torch.float64)
    ids = torch.tensor([[0, 1, 2, -1, -1], [3, 3, 4, 0, 1], [-1, 9, -1, -1, -1]])
    want = torch.stack([T[:3].mean(0), T[[3, 3, 4, 0, 1]].mean(0), T[0] * 0])
    got = MeanEmbedding(T).apply_batch(ids)
    assert got.dtype == torch.float64
    assert torch.allclose(got, want, rtol=0, atol=8 * 2.0 ** -53 * 20)
    est = EmbeddingClassifierEstimator(5, 3, dim=4, dropout=0.0)
    params = [p.double() for p in est.initial("cpu")]
    params[0] = T
    loss, _ = est.gradients(params, ids, torch.tensor([0, 1, 2]), 3, 1, 2)
    S = want @ params[1] + params[2]
    ref = torch.nn.functional.cross_entropy(S, torch.tensor([0, 1, 2]))
    assert abs(loss.item() - ref.item()) < 1e-14


@pytest.mark.skipif(not hip.available(), reason="extension not built")
def test_the_library_refuses_absent_memory():
    """Pointers that have to be there are checked before any launch: 1 is an
    invalid argument."""
    lib = hip._load()
    some = torch.zeros(4096, dtype=torch.uint8)
    p = some.data_ptr()

    def refused(name, args, absent):
        for i in absent:
            bad = list(args)
            assert bad[i] == p
            bad[i] = None
            assert getattr(lib, name)(*bad) == 1, (name, i)

    refused("ks_embedding_lookup", [p, 0, 3, p, 0, 5, 8, p, 8, 1.0, 4, None],
            (0, 3, 7))
    refused("ks_segment_sum", [1, p, 0, 2, 3, p, 0, 5, None, None, None, p, 0, 8,
                               p, 0, 8, None, 8, 1.0, 0, 4, None], (1, 5, 11, 14))
    refused("ks_segment_sum", [0, None, 9000, 1, 9000, p, 0, 5, None, None, None,
                               p, 0, 8, p, 0, 8, p, 8, 1.0, 0, 4, None], (17,))
    refused("ks_token_sort", [p, 0, 3, 5, 1, p, 0, 2, p, p, p, p, None, None],
            (0, 5, 8, 9, 11))
    refused("ks_token_sort", [p, 0, 9000, 5, 0, None, 1, 9000, p, p, None, p, p,
                              None], (12,))
    refused("ks_dropout", [p, p, 9, 0, 5, 1.0, 1, 2, None, None], (0, 1))
    refused("ks_fp8_quantise", [p, 0, 5, 3, 5, p, p, None], (0, 5, 6))
    refused("ks_fp8_linear", [p, 0, 5, p, p, None, p, 3, 5, 7, None, None],
            (0, 3, 4, 6))
    refused("ks_fp8_linear", [p, 0, 9000, p, p, None, p, 64, 9000, 700, p, None],
            (10,))


def test_no_kernel_runs_in_a_mode_of_fake_tensors():
    """Its results would have no memory either: refused before the launch."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        with pytest.raises(RuntimeError, match="memory"):
            hip._stream()
