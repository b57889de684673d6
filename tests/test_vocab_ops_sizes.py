"""The whole-vocabulary operators at sizes where one launch would need 2^32
threads: results are whole."""
import pytest
import torch

from glint_word2vec_amd.ops import fp8, softmax as S
from test_softmax_loss import U, _near, _reference

gpu = pytest.mark.gpu


@gpu
def test_gradient_of_more_than_2_30_numbers():
    """Two words, so that dh is p_0 (w_0 - w_1) up to its sign."""
    n, d = 1_050_000, 1024
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.empty(n, d, dtype=torch.bfloat16, device="cuda")
    for a in range(0, n, 150_000):
        h[a:a + 150_000] = torch.randn(150_000, d, generator=g,
                                       device="cuda") * 0.05
    w = torch.randn(2, d, generator=g, device="cuda").to(torch.bfloat16)
    y = torch.ones(n, dtype=torch.int32, device="cuda")
    loss, lse = S.softmax_loss_forward(h, w, y)
    dh, none = S.softmax_loss_backward(h, w, y, lse,
                                       torch.ones((), device="cuda"),
                                       need_w=False)
    for rows in (slice(0, 200), slice(n - 200, n)):
        want = _reference(h[rows], w, y[rows], grad=torch.ones(()))
        _near(dh[rows], want[4], want[6], "dh")


@gpu
def test_loss_of_more_than_2_26_rows():
    """Two words, one of them zeros: the loss is log(1 + exp(s)) of the score
    of the other."""
    n = (1 << 26) + 999
    h = torch.zeros(n, 2, dtype=torch.bfloat16, device="cuda")
    k = torch.arange(n, device="cuda") % 251
    h[:, 0] = (k - 125).to(torch.bfloat16) / 16
    w = torch.tensor([[1.0, 0.0], [0.0, 0.0]], dtype=torch.bfloat16,
                     device="cuda")
    y = torch.ones(n, dtype=torch.int32, device="cuda")
    loss, lse = S.softmax_loss_forward(h, w, y)
    want = torch.nn.functional.softplus(
        (torch.arange(251, device="cuda").double() - 125) / 16)[k]
    # the score is exact; two exponentials, their sum, a logarithm and its
    # product with log 2 remain, each of at most 8
    assert ((loss - want).abs() <= 8 * 16 * U).all()
    assert torch.equal(loss, lse)


@gpu
def test_8_bit_rows_of_more_than_2_30():
    n = (1 << 30) + 100
    x = torch.zeros(n, 1, dtype=torch.bfloat16, device="cuda")
    x[::3] = 1.5
    x[1::3] = -0.25
    q = fp8.quantize_rows(x)
    back = fp8.dequantize_rows(q, torch.bfloat16)
    assert torch.equal(back, x)
