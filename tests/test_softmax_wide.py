"""The forms of the kernels for much work, against float64: wide tiles of the
gradient's products, tiles of 256 x 256, and resident samples of 129 to 192
columns.  What is left out elsewhere since small work takes narrow tiles."""
import pytest
import torch

from glint_word2vec_amd.ops import fp8, softmax as S
from test_fp8_rows import _held, _product, _rows
from test_softmax_loss import U, _check, _inputs, _near, _reference

gpu = pytest.mark.gpu


# more than 4e9 products or 128 tiles: 4, 6, 8 and 10 blocks of 16 columns a
# wave for both gradients, and two tiles of them
@gpu
@pytest.mark.parametrize("n,v,d", [(1300, 33_000, 100), (800, 33_000, 160),
                                   (600, 33_000, 220), (450, 33_000, 300),
                                   (300, 33_001, 601)])
def test_bfloat16_gradients(n, v, d):
    _check(*_inputs(n, v, d, torch.bfloat16))


# more than 1e9 products, too few samples for parts of bfloat16: 6 and 10
# blocks for both, 8 for the table's
@gpu
@pytest.mark.parametrize("n,v,d", [(180, 31_000, 180), (180, 19_000, 300),
                                   (150, 20_000, 300)])
def test_float32_gradients(n, v, d):
    _check(*_inputs(n, v, d, torch.float32))


# 256 tiles of 256 x 256 and more
@gpu
@pytest.mark.parametrize("n,v,d", [(900, 20_000, 330), (1025, 13_057, 512)])
def test_large_tiles(n, v, d):
    _check(*_inputs(n, v, d, torch.bfloat16))


@gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(300, 40_000, 330), (1023, 16_390, 512)])
def test_large_tiles_of_8_bit_rows(m, n, k, out):
    b = _rows(n, k, torch.bfloat16, seed=m)
    cs = torch.rand(n, generator=torch.Generator().manual_seed(5)).cuda() + .5
    q, b64 = fp8.quantize_rows(b), _held(b)[0]
    a = _rows(m, k, torch.float32, seed=k)
    _product(a, q, b64, cs, out)
    _product(a, q, b64, out=out)


@gpu
@pytest.mark.parametrize("n,v,d", [(5, 400, 130), (16, 3000, 192),
                                   (64, 700, 150), (300, 3000, 190),
                                   (1000, 5000, 161)])
def test_resident_samples_of_six_steps(n, v, d):
    _check(*_inputs(n, v, d, torch.bfloat16))


@gpu
@pytest.mark.parametrize("n,v,d", [(256, 3000, 128), (40, 500, 400)])
def test_bfloat16_by_way_of_float32(n, v, d):
    """Gradients without coefficients in bfloat16, for who wants them: off by
    the last rounding alone, and by float32's."""
    h, w, y = _inputs(n, v, d, torch.bfloat16)
    a, b = h.requires_grad_(), w.requires_grad_()
    S.softmax_loss(a.float(), b.float(), y, reduction="sum").backward()
    assert a.grad.dtype == b.grad.dtype == torch.bfloat16
    r = _reference(a.detach().float(), b.detach().float(), y,
                   grad=torch.ones(()))
    _near(a.grad, r[4], r[6] + 2.0 ** -8 * (r[4].abs() + r[6]), "dh")
    _near(b.grad, r[5], r[7] + 2.0 ** -8 * (r[5].abs() + r[7]), "dw")
