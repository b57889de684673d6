"""What the whole-vocabulary operators leave of a model's and a table's state."""
import numpy as np
import pytest
import torch

from test_vocab_ops_model import _model, _tables

gpu = pytest.mark.gpu
U = 2.0 ** -24


@gpu
@pytest.mark.parametrize("count,alpha", [(40, 1e-3), (512, 5e-4)])
def test_repeated_centers_add_up_in_bfloat16(count, alpha):
    """Pairs of one center whose pushes are each under half a step of the row's
    entries: the sum of them moves it."""
    gs = _tables("bfloat16")
    c = torch.full((count + 8,), 7)
    c[:8] = torch.arange(20, 28)
    t = torch.full((count + 8,), 11)
    s0, s1 = gs.syn0[:, :52].double().cpu(), gs.syn1[:, :52].double().cpu()
    gs.train_softmax(c, t, alpha)
    p = torch.softmax(s0[c] @ s1.T, 1)
    p[:, 11] -= 1
    p = p * alpha
    add = torch.zeros_like(s0).index_add_(0, c, p @ s1)
    most = torch.zeros_like(s0).index_add_(0, c, p.abs() @ s1.abs())
    # a coefficient and its pair's gradient are rounded once each, with room
    # for the scores' error in float32; the row once, after the sum
    off = 3 * 2.0 ** -8 * most + 2.0 ** -8 * (s0 - add).abs() * 1.01
    got = gs.syn0[:, :52].double().cpu()
    assert ((got - (s0 - add)).abs() <= off).all()
    # (the row moves by far more than that)
    assert (add[7].abs() > 4 * off[7]).sum() > 20
    rest = [i for i in range(300) if i not in c.tolist()]
    assert torch.equal(got[rest], s0[rest])


@gpu
def test_model_loss_leaves_the_table_as_it_is():
    """A table that was trained on after to_gpu() is the one that the loss is
    of, and stays."""
    m = _model()
    m.to_gpu()
    sents = [["w0001", "w0005", "w0002"], ["w0003", "w0004"]]
    m._gpu.syn0 *= 2
    held = m._gpu.syn0.clone()
    s = (2 * torch.from_numpy(m.syn0)).double() @ \
        torch.from_numpy(m.syn1).double().T
    logp = torch.log_softmax(s, 1)
    pairs = [(1, 5), (5, 1), (5, 2), (2, 5), (1, 2), (2, 1), (3, 4), (4, 3)]
    want = -sum(float(logp[c, t]) for c, t in pairs) / len(pairs)
    for _ in range(2):
        assert m.softmax_loss(sents) == pytest.approx(
            want, abs=400 * U * float(s.abs().max() + 8))
        assert torch.equal(m._gpu.syn0, held)


class _Counting:
    """Stands for the device's tables: every pair's loss is its target."""
    device = torch.device("cpu")

    def __init__(self, text):
        self.text, self.sizes, self.read = text, [], []

    def softmax_loss(self, centers, targets):
        assert centers.shape == targets.shape
        self.sizes.append(len(centers))
        self.read.append(self.text.count)
        return targets.float()


class _Text:
    def __init__(self, sentences):
        self.sentences, self.count = sentences, 0

    def __iter__(self):
        for s in self.sentences:
            self.count += 1
            yield s


@pytest.mark.parametrize("batch", [1, 7, 64, 8192])
def test_model_loss_takes_the_text_a_batch_at_a_time(batch):
    """Pairs are made as they are needed: neither the text nor its pairs are
    held as a whole."""
    m = _model()
    rng = np.random.default_rng(1)
    sents = [[f"w{i:04d}" for i in rng.integers(0, 300, rng.integers(0, 9))]
             for _ in range(200)]
    text = _Text(sents)
    m._gpu, m._gpu_syn1 = _Counting(text), True
    got = m.softmax_loss(text, batch=batch)
    total = pairs = 0
    for s in sents:
        for i in range(len(s)):
            for j in range(len(s)):
                if i != j and abs(i - j) <= 3:
                    total, pairs = total + int(s[j][1:]), pairs + 1
    assert got == pytest.approx(total / pairs, rel=1e-12)
    assert sum(m._gpu.sizes) == pairs
    assert all(n == batch for n in m._gpu.sizes[:-1])
    assert 0 < m._gpu.sizes[-1] <= batch
    if batch < 100:
        assert m._gpu.read[0] < 40
