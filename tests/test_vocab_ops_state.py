"""What the whole-vocabulary operators leave of a model's and a table's state."""
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
