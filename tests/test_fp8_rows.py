"""Rows in 8-bit floats and their product, against plain float64 forms."""
import math

import pytest
import torch

from glint_word2vec_amd.ops import fp8

gpu = pytest.mark.gpu
U = 2.0 ** -24


def _held(x):
    """What rows stand for once they are held in 8 bits: (values, scales) in
    float64, from the definition."""
    x = x.double().cpu()
    r, k = x.shape
    out, scales = torch.zeros_like(x), []
    for c in range(0, k, 128):
        b = x[:, c:c + 128]
        finite = b.isfinite()
        most = torch.where(finite, b.abs(), 0.0).amax(1, keepdim=True)
        e = torch.ceil(torch.log2(most / 448)).clamp(-120, 120)
        u = b / torch.exp2(e)
        step = torch.exp2(torch.floor(torch.log2(u.abs())).clamp_min(-6) - 3)
        # at the largest scale values stop at 240: 256 * 2^120 is past float32
        u = torch.round(u / step) * step
        u = torch.where(e == 120, u.clamp(-240, 240), u)
        u = torch.where(finite, u, math.nan)
        out[:, c:c + 128] = u * torch.exp2(e)
        scales.append(torch.exp2(e))
    return out, torch.cat(scales, 1) if scales else x[:, :0]


def _rows(r, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(r, k, generator=g) * torch.exp(
        3 * torch.randn(r, 1, generator=g))
    return x.to(dtype).cuda()


SHAPES = [(1, 1), (1, 7), (3, 16), (2, 100), (5, 127), (4, 128), (7, 129),
          (33, 300), (130, 301), (9, 1024), (2, 2049), (1000, 64)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("r,k", SHAPES)
def test_quantize_is_exact(r, k, dtype):
    x = _rows(r, k, dtype, seed=r + k)
    q = fp8.quantize_rows(x)
    want, scales = _held(x)
    assert torch.equal(q.scales.float().double().cpu(), scales)
    assert torch.equal((q.values.float().cpu().double()
                        * scales.repeat_interleave(128, 1)[:, :k]), want)
    for out in (torch.float32, torch.bfloat16):
        back = fp8.dequantize_rows(q, out)
        assert back.dtype == out and torch.equal(back.double().cpu(), want)


@gpu
def test_quantize_edges():
    big, tiny = 3.3e38, 2.0 ** -140
    x = torch.zeros(10, 140)
    x[0, :3] = torch.tensor([448.0, 1.0, -0.0])       # scale 1
    x[1, :2] = torch.tensor([448.0001, 8.5])          # scale 2
    x[2, :2] = torch.tensor([big, 1.0])
    x[3, :2] = torch.tensor([tiny, -tiny])            # below the least scale
    x[4, :3] = torch.tensor([math.nan, 1.0, 2.0])
    x[5, :3] = torch.tensor([math.inf, -math.inf, 5.0])
    x[6] = math.nan
    x[7, 128:] = 2.0 ** -120 * 448
    x[8, :2] = torch.tensor([1.0625 * 16, 1.1875 * 16])   # ties, at scale 2^-4
    x[9, 139] = -17.0
    q = fp8.quantize_rows(x.cuda())
    want, scales = _held(x)
    assert torch.equal(q.scales.float().double().cpu(), scales)
    got = fp8.dequantize_rows(q).double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    # behind the last column, up to 16 bytes, are zeros
    held = q.values.as_strided((10, 144), (144, 1)).view(torch.uint8)
    assert (held[:, 140:] == 0).all()


@gpu
def test_quantize_error_is_half_a_step():
    x = _rows(50, 256, torch.float32)
    q = fp8.quantize_rows(x)
    off = (fp8.dequantize_rows(q) - x).abs()
    s = q.scales.float().repeat_interleave(128, 1)
    assert (off <= torch.maximum(x.abs() * 2 ** -4, s * 2 ** -10)).all()


@gpu
def test_strides():
    big = torch.full((40, 400), math.nan, device="cuda")
    big[1:31, 3:303] = _rows(30, 300, torch.float32)
    x = big[1:31, 3:303]
    want, _ = _held(x)
    for t in (x, x.T.contiguous().T, x.contiguous()):
        assert torch.equal(fp8.dequantize_rows(
            fp8.quantize_rows(t)).double().cpu(), want)
    q = fp8.quantize_rows(x)
    # rows of the held table that start anywhere, and every other one
    odd = torch.full((30, 317), 0x7f, dtype=torch.uint8, device="cuda")
    odd[:, 5:305] = q.values.view(torch.uint8)
    odd = fp8.Fp8Rows(odd.view(torch.float8_e4m3fn)[:, 5:305], q.scales)
    assert torch.equal(fp8.dequantize_rows(odd).double().cpu(), want)
    some = fp8.Fp8Rows(q.values[::2], q.scales[::2])
    assert torch.equal(fp8.dequantize_rows(some).double().cpu(), want[::2])
    a = _rows(5, 300, torch.float32, seed=4)
    _product(a, odd, want)
    _product(a, some, want[::2])


def _product(a, b, b64, col_scale=None, out=torch.float32, given=False):
    a64, _ = _held(a)
    k = a.shape[1]
    want = a64 @ b64.T
    off = (k + 2) * U * 2 * (a64.abs() @ b64.abs().T)
    if col_scale is not None:
        cs = col_scale.double().cpu()
        want, off = want * cs, off * cs.abs() + U * 2 * (want * cs).abs()
    step = 2.0 ** -8 if out == torch.bfloat16 else U
    off = off + step * (want.abs() + off) + 1e-38
    got = fp8.matmul_rows(fp8.quantize_rows(a) if given else a, b,
                          col_scale=col_scale, out_dtype=out)
    assert got.dtype == out and got.shape == want.shape
    got = got.double().cpu()
    bad = ~((got - want).abs() <= off)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off"


# (queries at which another kernel takes over, narrow and wide rows)
PRODUCTS = [(16, 700, 20), (17, 700, 321), (16, 300, 2049), (32, 1025, 330),
            (40, 600, 64), (160, 300, 400), (161, 515, 400), (200, 900, 321),
            (300, 601, 200), (2, 150_000, 40), (70, 70_001, 300),
            (18, 150_000, 330), (1, 1, 1), (1, 5, 16), (1, 300, 300), (2, 129, 128), (16, 1000, 100),
            (17, 257, 301), (33, 64, 1024), (64, 500, 257), (65, 128, 640),
            (128, 3613, 100), (129, 130, 131), (300, 700, 2048)]


@gpu
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, out):
    b = _rows(n, k, torch.bfloat16, seed=m + n)
    cs = torch.rand(n, generator=torch.Generator().manual_seed(5)).cuda() + .5
    q, b64 = fp8.quantize_rows(b), _held(b)[0]
    a = _rows(m, k, torch.float32, seed=k)
    _product(a, q, b64, out=out)
    _product(a, q, b64, cs, out)
    _product(a.bfloat16(), q, b64, cs, out)
    _product(a, q, b64, cs, out, given=True)


@gpu
@pytest.mark.parametrize("m", [1, 20, 161])
def test_widest_product(m):
    """2^20 columns; more are refused."""
    k = 1 << 20
    b = _rows(70, k, torch.bfloat16)
    _product(_rows(m, k, torch.bfloat16, seed=1), fp8.quantize_rows(b),
             _held(b)[0])
    with pytest.raises(ValueError, match="2\\^20"):
        fp8.matmul_rows(torch.zeros(1, k + 1, device="cuda"),
                        fp8.quantize_rows(torch.zeros(1, k + 1,
                                                      device="cuda")))


@gpu
def test_product_in_many_pieces(monkeypatch):
    """More table rows than one piece of the converted table holds."""
    b = _rows(9000, 4000, torch.bfloat16, seed=3)
    q, b64 = fp8.quantize_rows(b), _held(b)[0]
    cs = torch.rand(9000, generator=torch.Generator().manual_seed(5)).cuda()
    _product(_rows(170, 4000, torch.float32), q, b64, cs, torch.bfloat16)


@gpu
def test_scales_that_start_anywhere():
    b = _rows(200, 300, torch.float32)
    q, b64 = fp8.quantize_rows(b), _held(b)[0]
    for before in (1, 2, 3):
        flat = torch.zeros(200 * 3 + before, dtype=torch.uint8, device="cuda")
        flat[before:] = q.scales.view(torch.uint8).flatten()
        moved = fp8.Fp8Rows(q.values, flat[before:].view(200, 3)
                            .view(torch.float8_e8m0fnu))
        for m in (1, 20, 80):
            _product(_rows(m, 300, torch.float32, m), moved, b64)
    wide = torch.zeros(200, 5, dtype=torch.uint8, device="cuda")
    wide[:, 1:4] = q.scales.view(torch.uint8)
    moved = fp8.Fp8Rows(q.values, wide.view(torch.float8_e8m0fnu)[:, 1:4])
    _product(_rows(20, 300, torch.float32), moved, b64)
    assert torch.equal(fp8.dequantize_rows(moved).double().cpu(), b64)


@gpu
def test_product_of_extreme_scales():
    """Blocks of one row whose scales lie 2^40 apart."""
    b = torch.randn(200, 384, generator=torch.Generator().manual_seed(1))
    b[:, 128:256] *= 2.0 ** 20
    b[:, 256:] *= 2.0 ** -20
    b = b.cuda()
    a = b[:20].flip(1).contiguous()
    _product(a, fp8.quantize_rows(b), _held(b)[0])
    z = torch.zeros(3, 384, device="cuda")
    assert (fp8.matmul_rows(z, fp8.quantize_rows(b)) == 0).all()


@gpu
def test_rows_that_are_not_finite_stay_alone():
    a, b = _rows(20, 150, torch.float32), _rows(300, 150, torch.float32, 1)
    a[3, 7], b[299, 140], b[5, 0] = math.nan, math.inf, math.nan
    out = fp8.matmul_rows(a, fp8.quantize_rows(b)).cpu()
    want = torch.zeros(20, 300, dtype=torch.bool)
    want[3], want[:, 299], want[:, 5] = True, True, True
    assert torch.equal(out.isnan(), want)


@gpu
def test_empty():
    b = fp8.quantize_rows(_rows(10, 20, torch.float32))
    assert fp8.matmul_rows(torch.zeros(0, 20).cuda(), b).shape == (0, 10)
    none = fp8.quantize_rows(torch.zeros(0, 20).cuda())
    assert none.shape == (0, 20) and none.scales.shape == (0, 1)
    assert fp8.dequantize_rows(none).shape == (0, 20)
    assert fp8.matmul_rows(torch.ones(3, 20).cuda(), none).shape == (3, 0)
    assert fp8.matmul_rows(none, b).shape == (0, 10)


@gpu
def test_streams_and_graphs():
    a, b = _rows(9, 200, torch.float32), _rows(700, 200, torch.float32, 1)
    first = fp8.matmul_rows(a, fp8.quantize_rows(b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = fp8.matmul_rows(a, fp8.quantize_rows(b))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    sa, sb = a.clone(), b.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fp8.matmul_rows(sa, fp8.quantize_rows(sb))
    for k in range(3):
        sa.copy_(_rows(9, 200, torch.float32, 10 + k))
        sb.copy_(_rows(700, 200, torch.float32, 20 + k))
        graph.replay()
        want = fp8.matmul_rows(sa.clone(), fp8.quantize_rows(sb.clone()))
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@gpu
def test_output_past_32_bits():
    """More than 2^31 scores: the last rows are right."""
    m, n, k = 2100, 1_050_000, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    b = fp8.quantize_rows(torch.randn(n, k, generator=g, device="cuda"))
    a = torch.randn(m, k, generator=g, device="cuda")
    out = fp8.matmul_rows(a, b)
    part = fp8.dequantize_rows(b)
    a64 = _held(a[-3:])[0].cuda()
    want = a64 @ part.double().T
    off = (k + 3) * U * 2 * (a64.abs() @ part.double().abs().T) + 1e-38
    assert ((out[-3:] - want).abs() <= off).all()


def test_refusals():
    x = torch.zeros(4, 8)
    for bad, error in (([1.0], TypeError), (x[0], ValueError),
                       (x[:, :0], ValueError), (x.half(), TypeError),
                       (x.int(), TypeError), (x, RuntimeError)):
        with pytest.raises(error):
            fp8.quantize_rows(bad)
    values = torch.zeros(4, 8, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    good = fp8.Fp8Rows(values, scales)
    for bad, error in ((x, TypeError), ((values, scales), TypeError),
                       (fp8.Fp8Rows(x, scales), TypeError),
                       (fp8.Fp8Rows(values, x[:, :1]), TypeError),
                       (fp8.Fp8Rows(values, scales[:3]), ValueError),
                       (fp8.Fp8Rows(values[0], scales), ValueError),
                       (good, RuntimeError)):
        with pytest.raises(error):
            fp8.dequantize_rows(bad)
        with pytest.raises(error):
            fp8.matmul_rows(x, bad)


@gpu
def test_refusals_of_the_product():
    b = fp8.quantize_rows(_rows(10, 20, torch.float32))
    a = torch.zeros(2, 20, device="cuda")
    cs = torch.zeros(10, device="cuda")
    for kw, error in ((dict(a=a[:, :19]), ValueError),
                      (dict(a=a.cpu()), RuntimeError),
                      (dict(a=a.half()), TypeError),
                      (dict(out_dtype=torch.float16), TypeError),
                      (dict(col_scale=cs[:9]), ValueError),
                      (dict(col_scale=cs.double()), ValueError),
                      (dict(col_scale=1.0), TypeError),
                      (dict(col_scale=cs.cpu()), RuntimeError)):
        with pytest.raises(error):
            fp8.matmul_rows(**{"a": a, "b": b, **kw})
    with pytest.raises(TypeError):
        fp8.dequantize_rows(b, torch.float16)
