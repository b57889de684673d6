"""The operators over the whole vocabulary as the tables and models use them."""
import numpy as np
import pytest
import torch

from glint_word2vec_amd.config import Word2VecConfig
from glint_word2vec_amd.estimator import GlintWord2VecModel
from glint_word2vec_amd.vocab import Vocabulary

gpu = pytest.mark.gpu
U = 2.0 ** -24


def _model(vocab=300, dim=52, seed=0, window=3):
    rng = np.random.default_rng(seed)
    words = [f"w{i:04d}" for i in range(vocab)]
    voc = Vocabulary(words=words, counts=np.ones(vocab, dtype=np.int64),
                     index={w: i for i, w in enumerate(words)},
                     train_words_count=vocab)
    syn0 = rng.standard_normal((vocab, dim)).astype(np.float32)
    syn1 = rng.standard_normal((vocab, dim)).astype(np.float32) * 0.3
    return GlintWord2VecModel(Word2VecConfig(vector_size=dim, window=window),
                              voc, syn0, syn1)


def _tables(dtype, vocab=300, dim=52):
    from glint_word2vec_amd.ops.gpu import GpuSgns
    m = _model(vocab, dim)
    gs = GpuSgns(vocab, dim, dtype=dtype, device="cuda")
    gs.load_host(m.syn0 * 0.3, m.syn1)
    return gs


def _held(x):
    """float64 values that rows of columns <= 128 stand for in 8 bits."""
    x = x.double()
    e = torch.ceil(torch.log2(x.abs().amax(1, keepdim=True) / 448))
    u = x / torch.exp2(e)
    step = torch.exp2(torch.floor(torch.log2(u.abs())).clamp_min(-6) - 3)
    return torch.round(u / step) * step * torch.exp2(e)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_softmax_step(dtype):
    """One step against the formula in float64, with repeated centers and
    targets that are cut off."""
    gs = _tables(dtype)
    g = torch.Generator().manual_seed(2)
    c = torch.randint(0, 40, (150,), generator=g)
    t = torch.randint(0, 300, (150,), generator=g, dtype=torch.int32)
    t[::7] = -1
    s0, s1 = gs.syn0[:, :52].double().cpu(), gs.syn1[:, :52].double().cpu()
    alpha = 0.05
    loss = gs.train_softmax(c.cuda(), t.cuda(), alpha)
    kept = t >= 0
    s = s0[c] @ s1.T
    logp = torch.log_softmax(s, 1)
    want = torch.where(kept, -logp[torch.arange(150), t.long().clamp_min(0)],
                       0.0)
    # scores are sums of 52 products of about 0.1, 60 U off at most; the sum
    # over 300 words and two logarithms add as much
    assert (loss.double().cpu() - want).abs().max() < 400 * U * (
        s.abs().max() + 8)
    p = logp.exp()
    p[torch.arange(150), t.long().clamp_min(0)] -= 1
    p = p * kept[:, None] * alpha
    d0, d1 = p @ s1, p.T @ s0[c]
    half = 2.0 ** -8 if dtype == "bfloat16" else U
    # coefficients, gradients and the tables are each rounded once, and sums
    # of n terms n times in float32; the probabilities are 64 U (|s| + 8) off
    rel = half * 3 + 400 * U * (float(s.abs().max()) + 8)
    off1 = rel * (p.abs().T @ s0[c].abs()) + half * (
        d1.abs() + (s1 - d1).abs()) * 1.01
    add0 = torch.zeros_like(s0).index_add_(0, c, d0)
    most0 = torch.zeros_like(s0).index_add_(0, c, p.abs() @ s1.abs())
    count = torch.bincount(c, minlength=300)[:, None].double()
    off0 = rel * most0 * 2 + half * (s0.abs() + most0) * (count > 0) * 1.01 \
        + 4 * count * U * (s0.abs() + most0)
    assert ((gs.syn1[:, :52].double().cpu() - (s1 - d1)).abs() <= off1).all()
    assert ((gs.syn0[:, :52].double().cpu() - (s0 - add0)).abs() <= off0).all()
    # what lies behind the last column stays zero
    assert (gs.syn0[:, 52:] == 0).all() and (gs.syn1[:, 52:] == 0).all()


@gpu
def test_softmax_step_is_the_same_on_every_run():
    a, b = _tables("bfloat16"), _tables("bfloat16")
    g = torch.Generator().manual_seed(2)
    c = torch.randint(0, 20, (500,), generator=g)
    t = torch.randint(0, 300, (500,), generator=g)
    for _ in range(3):
        assert torch.equal(a.train_softmax(c, t, 0.05),
                           b.train_softmax(c, t, 0.05))
    assert torch.equal(a.syn0, b.syn0) and torch.equal(a.syn1, b.syn1)


@gpu
def test_pairs_that_are_no_words():
    """They move nothing, and the other pairs as if they were not there."""
    a, b = _tables("float32"), _tables("float32")
    c = torch.tensor([3, -1, 300, 7, 2 ** 40, -1, 3, 9])
    t = torch.tensor([5, 6, 7, 300, 8, -1, -1, 11])
    want = a.softmax_loss(c[[0, 7]], t[[0, 7]])
    for gs in (a, b):
        got = gs.softmax_loss(c, t) if gs is a else \
            gs.train_softmax(c, t, 0.1)
        assert got[[1, 2, 3, 4]].isnan().all()
        assert (got[[5, 6]] == 0).all()
        assert torch.equal(got[[0, 7]], want)
    good = _tables("float32")
    good.train_softmax(c[[0, 7]], t[[0, 7]], 0.1)
    # sums over eight pairs and over two may be cut differently: within the
    # rounding of two products of one step
    for x, y in ((b.syn0, good.syn0), (b.syn1, good.syn1)):
        assert (x - y).abs().max() <= 64 * U * float(y.abs().max())
    assert torch.equal(b.syn0[4:9:4], _tables("float32").syn0[4:9:4])
    with pytest.raises(ValueError, match="centers"):
        a.softmax_loss(c, t[:3])


@gpu
def test_step_then_loss_then_8_bit_scores():
    """The operators one after the other, as a program trains on the whole
    softmax and answers from 8 bits: each against the tables as they are."""
    gs = _tables("bfloat16")
    g = torch.Generator().manual_seed(4)
    c = torch.randint(0, 300, (200,), generator=g)
    t = torch.randint(0, 300, (200,), generator=g)
    gs.train_softmax(c, t, 0.1)
    s0, s1 = gs.syn0[:, :52].double().cpu(), gs.syn1[:, :52].double().cpu()
    s = s0[c] @ s1.T
    want = -torch.log_softmax(s, 1)[torch.arange(200), t]
    got = gs.softmax_loss(c.cuda(), t.cuda()).double().cpu()
    assert (got - want).abs().max() < 400 * U * (s.abs().max() + 8)
    table, norms = gs.quantize_table(), gs.norms()
    q = torch.randn(9, 52, generator=g)
    got = gs.multiply_fp8(q, table, norms).double().cpu()
    a, b = _held(q), _held(s0)
    n = s0.norm(dim=1)
    off = 120 * U * (a.abs() @ b.abs().T) / n + 64 * U * (a @ b.T / n).abs()
    assert ((got - a @ b.T / n).abs() <= off).all()
    assert torch.equal(gs.multiply_fp8(q, table),
                       gs.multiply_fp8(q.cuda(), table, None))


@gpu
def test_model_loss():
    m = _model()
    sents = [["w0001", "w0005", "w0002", "unknown", "w0009"], ["w0007"], [],
             ["w0003", "w0003"]]
    with pytest.raises(RuntimeError):
        m.softmax_loss(sents)
    m.to_gpu()
    pairs = []
    for ids in ([1, 5, 2, 9], [3, 3]):
        pairs += [(ids[i], ids[j]) for i in range(len(ids))
                  for j in range(len(ids)) if i != j and abs(i - j) <= 3]
    c, t = torch.tensor(pairs).T
    s = torch.from_numpy(m.syn0).double()[c] @ \
        torch.from_numpy(m.syn1).double().T
    want = float(-torch.log_softmax(s, 1)[torch.arange(len(c)), t].mean())
    for batch in (5, 8192):
        assert m.softmax_loss(sents, batch=batch) == pytest.approx(
            want, abs=400 * U * float(s.abs().max() + 8))
    assert np.isnan(m.softmax_loss([["w0001"]]))
    m.syn1 = None
    with pytest.raises(ValueError):
        m.softmax_loss(sents)


@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_synonyms_from_8_bits(dtype):
    """The words and cosines of the 8-bit table's own values."""
    m = _model()
    m.syn0[17] = 0
    m.to_gpu(dtype=dtype, scores="fp8")
    s0 = torch.from_numpy(m.syn0)
    if dtype == "bfloat16":
        s0 = s0.bfloat16().float()
    rows = _held(s0)
    rows[17] = 0
    n = s0.double().norm(dim=1)
    asked = ["w0003", "w0100", m.syn0[5] * 2]
    vecs = np.stack([m.syn0[3], m.syn0[100], m.syn0[5] * 2])
    q = vecs / np.linalg.norm(vecs, axis=1, keepdims=True)
    cos = _held(torch.from_numpy(q)) @ rows.T / n
    cos[:, 17] = 0
    batch = m.find_synonyms_batch(asked, 5)
    one = [m.find_synonyms(a, 5) for a in asked]
    for i, a in enumerate(asked):
        order = [j for j in cos[i].argsort(descending=True).tolist()
                 if not (isinstance(a, str) and m.vocab.words[j] == a)][:5]
        for got in (batch[i], one[i]):
            assert [w for w, _ in got] == [m.vocab.words[j] for j in order]
            for (_, v), j in zip(got, order):
                # 52 terms of at most 1 in all, and the norm
                assert v == pytest.approx(float(cos[i, j]), abs=200 * U)


@gpu
def test_sharded_synonyms_from_8_bits(tmp_path):
    m = _model()
    m.save(str(tmp_path / "m"), num_shards=3)
    sharded = GlintWord2VecModel.load_sharded(
        str(tmp_path / "m"), device="cuda", dtype="float32", scores="fp8")
    m.to_gpu(scores="fp8")
    asked = ["w0003", "w0250", m.syn0[9]]
    for a, b in zip(sharded.find_synonyms_batch(asked, 7),
                    m.find_synonyms_batch(asked, 7)):
        assert [w for w, _ in a] == [w for w, _ in b]
        assert [v for _, v in a] == pytest.approx([v for _, v in b],
                                                  abs=200 * U)


def test_refusals(tmp_path):
    m = _model()
    with pytest.raises(ValueError):
        m.to_gpu(scores="int8")
    with pytest.raises(RuntimeError):
        m.softmax_loss([["w0001", "w0002"]])
    with pytest.raises(ValueError, match="batch"):
        m.softmax_loss([["w0001", "w0002"]], batch=0)
    m.save(str(tmp_path / "m"))
    with pytest.raises(ValueError):
        GlintWord2VecModel.load_sharded(str(tmp_path / "m"), device="cpu",
                                        scores="int8")
    with pytest.raises(RuntimeError):
        GlintWord2VecModel.load_sharded(str(tmp_path / "m"), device="cpu",
                                        scores="fp8")
