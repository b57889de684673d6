"""What the whole-vocabulary operators leave of a model's and a table's state."""
import numpy as np
import pytest
import torch

from test_vocab_ops_model import _model, _tables

gpu = pytest.mark.gpu
U = 2.0 ** -24


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
