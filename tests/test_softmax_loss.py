"""Softmax cross entropy over the whole vocabulary against a plain float64
form.  Tolerances count roundings: a product's sum of D terms in float32 is off
by at most D * 2^-24 of the sum of absolute terms, a stored number by half a
step of its type."""
import math

import pytest
import torch

from glint_word2vec_amd.ops import softmax as S

gpu = pytest.mark.gpu
U = 2.0 ** -24


def _inputs(n, v, d, dtype, seed=0, spread=1.5, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(n, d, generator=g) * spread / d ** 0.25
    w = torch.randn(v, d, generator=g) * spread / d ** 0.25
    y = torch.randint(0, v, (n,), generator=g)
    return h.to(dtype).to(device), w.to(dtype).to(device), y.to(device)


def _reference(h, w, y, ignore=-1, grad=None):
    """Loss, lse, dh, dw of sum grad_n loss_n in float64, and how far the
    kernels' may be from them."""
    bf16 = h.dtype == torch.bfloat16
    h, w, y = h.double().cpu(), w.double().cpu(), y.long().cpu()
    n, d = h.shape
    v = w.shape[0]
    s = h @ w.T
    # one score: d roundings of the running sum, and the products' own in f32
    off_s = 2 * (d + 2) * U * (h.abs() @ w.abs().T)
    lse = torch.logsumexp(s, 1)
    # the sum over the vocabulary: every lane adds v / 8 terms or fewer, its
    # exponentials are off by 2 steps and by the score's error
    most = off_s.amax(1) if n else off_s.new_zeros(0)
    off_lse = most + (v / 8 + 64) * U + 8 * U * (lse.abs() + 1) \
        + 4 * U * s.abs().amax(1)
    kept = y != ignore
    yy = y.clamp(0, v - 1)
    loss = torch.where(kept, lse - s.gather(1, yy[:, None])[:, 0], 0.0)
    off_loss = off_lse + most + 2 * U * loss.abs()
    if grad is None:
        return loss, lse, off_loss, off_lse
    grad = grad.double().cpu().expand(n) * kept
    p = torch.exp(s - lse[:, None])
    c = p.clone()
    c[torch.arange(n), yy] -= 1
    c = c * grad[:, None]
    off_c = p * grad.abs()[:, None] * (
        2 * (off_s + off_lse[:, None]) + 16 * U) + 4 * U * c.abs()
    if bf16:
        off_c = off_c + 2.0 ** -8 * (c.abs() + off_c)
    step = 2.0 ** -8 if bf16 else U
    dh, dw = c @ w, c.T @ h
    off_dh = (off_c + 2 * (v + 2) * U * c.abs()) @ w.abs()
    off_dw = (off_c + 2 * (n + 2) * U * c.abs()).T @ h.abs()
    off_dh = off_dh + step * (dh.abs() + off_dh) + 1e-38
    off_dw = off_dw + step * (dw.abs() + off_dw) + 1e-38
    return loss, lse, off_loss, off_lse, dh, dw, off_dh, off_dw


def _near(got, want, off, what):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = (got - want).abs() > off
    bad |= got.isnan()
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
        f"{float(((got - want).abs() / off).max()):.3g} of the tolerance")


def _check(h, w, y, ignore=-1, seed=1):
    g = torch.randn(len(h), generator=torch.Generator().manual_seed(seed))
    g = g.to(h.device)
    loss, lse, ol, oe, dh, dw, oh, ow = _reference(h, w, y, ignore, g)
    got, got_lse = S.softmax_loss_forward(h, w, y, ignore_index=ignore)
    _near(got, loss, ol, "loss")
    _near(got_lse, lse, oe, "lse")
    a, b = S.softmax_loss_backward(h, w, y, got_lse, g, ignore_index=ignore)
    assert a.dtype == h.dtype and b.dtype == w.dtype
    _near(a, dh, oh, "dh")
    _near(b, dw, ow, "dw")


SHAPES = [(1, 1, 1), (1, 2, 3), (2, 127, 8), (3, 128, 100), (1, 129, 301),
          (127, 129, 64), (128, 256, 128), (129, 257, 300), (17, 1000, 520),
          (200, 3613, 100), (300, 5000, 65), (64, 777, 1024), (5, 300, 2048)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,d", SHAPES)
def test_matches_float64(n, v, d, dtype):
    _check(*_inputs(n, v, d, dtype, seed=n + v + d))


# samples around the sizes at which another kernel takes over, narrow and wide
# rows
FORMS = [(16, 700, 20), (17, 700, 321), (32, 1025, 330), (33, 600, 400),
         (64, 900, 640), (65, 513, 321), (100, 1300, 512), (128, 1000, 40),
         (130, 1000, 700), (256, 2600, 200), (300, 515, 1030), (31, 257, 2049),
         (700, 300, 33)]


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,d", FORMS)
def test_forms(n, v, d, dtype):
    _check(*_inputs(n, v, d, dtype, seed=n + v + d))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,d", [(2, 150_000, 24), (40, 150_001, 300),
                                   (40, 140_000, 330), (260, 70_000, 40)])
def test_many_tiles_for_each_workgroup(n, v, d, dtype):
    _check(*_inputs(n, v, d, dtype))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [5, 70])
def test_many_pieces_of_the_vocabulary(n, dtype, monkeypatch):
    monkeypatch.setattr(S, "_COEF_BYTES", 1 << 16)
    monkeypatch.setattr(S, "_PACKED_BYTES", 1 << 16)
    h, w, y = _inputs(n, 1500, 97, dtype)
    _check(h, w, y)
    # unaligned, so that the pieces are packed
    big = torch.zeros(1502, 103, dtype=dtype, device="cuda")
    big[1:-1, 5:102] = w
    _check(h, big[1:-1, 5:102], y)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_offsets(dtype):
    """Padded rows with NaN behind the last column and above and below the
    rows, odd starts, and columns that are not neighbours."""
    n, v, d = 37, 200, 75
    h, w, y = _inputs(n, v, d, dtype)

    def inside(t, before, after):
        big = torch.full((t.shape[0] + 2, t.shape[1] + before + after),
                         math.nan, dtype=t.dtype, device=t.device)
        big[1:-1, before:before + t.shape[1]] = t
        return big[1:-1, before:before + t.shape[1]]
    for before, after in ((0, 5), (0, 6), (8, 5), (1, 4), (3, 0)):
        _check(inside(h, before, after), inside(w, before, after), y)
    _check(h.T.contiguous().T, w.T.contiguous().T, y)
    _check(h[::2], w, y[::2])
    _check(h, w.flip(0)[::3], y % 67)
    _check(h[:1].expand(n, d), w, y)


@pytest.fixture
def in_parts(monkeypatch):
    """float32 of any size in parts of bfloat16."""
    monkeypatch.setattr(S, "_SPLIT_LOSS", (0, 0))
    monkeypatch.setattr(S, "_SPLIT_GRAD", (0, 0))


@gpu
@pytest.mark.parametrize("n,v,d", SHAPES + FORMS + [(260, 70_000, 40)])
def test_parts_of_bfloat16(n, v, d, in_parts):
    """As exact as float32: the same tolerances."""
    _check(*_inputs(n, v, d, torch.float32, seed=n + v + d))


@gpu
@pytest.mark.parametrize("n,v,d", [(384, 60_000, 100), (192, 56_000, 100),
                                   (191, 56_300, 100), (383, 60_000, 100)])
def test_where_parts_begin(n, v, d):
    """Sizes at which the form changes, as they are chosen."""
    _check(*_inputs(n, v, d, torch.float32))


@gpu
@pytest.mark.parametrize("n,v,d", [(285, 95, 588), (192, 56_000, 100),
                                   (600, 20_000, 96)])
def test_gradient_from_scores_rounded_alike(n, v, d):
    """Confident rows, whose targets score 12 and the other words little.
    Where a target's score and those in lse are rounded alike, an error e_v of
    the scores changes p_v by p_v (e_v - sum_k p_k e_k): for the target, whose
    p is almost 1, by 2 p (1 - p) of the largest.  What is left is lse in
    float32, its product with log2 e and the exponent's own rounding: (3 |lse|
    + 3 |s|) U, and with the sum's and the exponentials' roundings twice
    that and (v / 8 + 64) U (1 - p), 16 U at most."""
    g = torch.Generator().manual_seed(n)
    w = torch.randn(v, d, generator=g)
    y = torch.randint(0, v, (n,), generator=g)
    h = w[y] * (12.0 / (w[y] ** 2).sum(1, keepdim=True))
    h = h + 0.3 * torch.randn(n, d, generator=g) / d ** 0.5
    a, b = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    S.softmax_loss(a, b, y.cuda(), reduction="sum").backward()
    _, lse = S.softmax_loss_forward(h.cuda(), w.cuda(), y.cuda(),
                                    gradient=True)
    pair = S.softmax_loss_backward(h.cuda(), w.cuda(), y.cuda(), lse,
                                   torch.ones((), device="cuda"))
    h, w = h.double(), w.double()
    s = h @ w.T
    off_s = (2 * (d + 2) * U * (h.abs() @ w.abs().T)).amax(1, keepdim=True)
    p = torch.softmax(s, 1)
    lse = torch.logsumexp(s, 1, keepdim=True)
    c = p.clone()
    c[torch.arange(n), y] -= 1
    off_c = p * (2 * (1 - p) * off_s * 1.01 + (1 - p) * (v / 8 + 64) * U
                 + 6 * U * (lse.abs() + s.abs()) + 16 * U) + 4 * U * c.abs()
    dh, dw = c @ w, c.T @ h
    off_dh = (off_c + 2 * (v + 2) * U * c.abs()) @ w.abs() + 2 * U * dh.abs()
    off_dw = (off_c + 2 * (n + 2) * U * c.abs()).T @ h.abs() \
        + 2 * U * dw.abs()
    for x, z in ((a.grad, b.grad), pair):
        _near(x, dh, off_dh, "dh")
        _near(z, dw, off_dw, "dw")


@gpu
@pytest.mark.parametrize("n", [3, 40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widest_rows(n, dtype):
    """2^20 columns; more are refused."""
    _check(*_inputs(n, 70, 1 << 20, dtype))


@gpu
def test_widest_rows_in_parts(in_parts):
    _check(*_inputs(5, 70, 1 << 20, torch.float32))


@gpu
def test_parts_of_every_magnitude(in_parts, monkeypatch):
    """Numbers from 2^-126 up to float32's largest, alone in their rows, so
    that each score is one product: within two roundings of it, and within a
    subnormal part of bfloat16 (2^-134) times the other factor."""
    monkeypatch.setattr(S, "_COEF_BYTES", 1 << 16)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(300, 1, generator=g)
    x = x / x.abs() * 2.0 ** torch.linspace(-126, 127.99, 300)[:, None]
    x[-1] = torch.finfo(torch.float32).max
    h = torch.zeros(300, 40)
    h[:, 7] = x[:, 0]
    w = torch.zeros(2, 40)
    for f in (1.0, 1 + 2.0 ** -8 + 2.0 ** -16 + 2.0 ** -23, 2.0 ** -100,
              -0.99999994):
        w[0, 7] = f
        want = h[:, 7].double() * float(w[0, 7])
        # a product past float32 is not finite in any form
        fits = want.abs() <= torch.finfo(torch.float32).max
        y = torch.ones(300, dtype=torch.long, device="cuda")
        # the loss of word 1, whose score is 0, is log(1 + exp(score)): the
        # score itself where that is large
        loss, lse = S.softmax_loss_forward(h.cuda(), w.cuda(), y)
        ref = torch.logaddexp(want, torch.zeros_like(want))
        off = 4 * U * want.abs() + 2.0 ** -134 * abs(float(w[0, 7])) + 8 * U
        assert ((loss.double().cpu() - ref).abs() <= off)[fits].all()
        assert fits.sum() >= 299
    # and as gradients: one sample, whose coefficients are p - 1 = -1/2
    for rows in x.reshape(-1, 10)[:29]:
        h = rows[:, None].repeat(1, 40).cuda()
        dh, dw = S.softmax_loss_backward(
            h, torch.zeros(2, 40, device="cuda"),
            torch.zeros(10, dtype=torch.long, device="cuda"),
            torch.full((10,), math.log(2.0), device="cuda"),
            torch.ones((), device="cuda"))
        assert (dh == 0).all()
        want = -0.5 * rows.double().sum()
        off = 16 * U * rows.double().abs().sum() + 2.0 ** -133
        assert ((dw[0].double().cpu() - want).abs() <= off).all()


@gpu
def test_parts_strides_ignored_and_not_finite(in_parts, monkeypatch):
    monkeypatch.setattr(S, "_COEF_BYTES", 1 << 16)
    monkeypatch.setattr(S, "_PACKED_BYTES", 1 << 16)
    h, w, y = _inputs(100, 1500, 97, torch.float32)
    big_h = torch.full((100, 203), math.nan, device="cuda")
    big_h[:, 5:199:2] = h
    big_w = torch.full((1502, 103), math.nan, device="cuda")
    big_w[1:-1, 5:102] = w
    y[::9] = -1
    _check(big_h[:, 5:199:2], big_w[1:-1, 5:102], y)
    one = torch.ones((), device="cuda")
    good, lse = S.softmax_loss_forward(h, w, y)
    dh, dw = S.softmax_loss_backward(h, w, y, lse, one)
    # rows without a loss may hold anything
    h[::9] = math.nan
    h[0], h[9] = math.inf, -math.inf
    loss, lse = S.softmax_loss_forward(h, w, y)
    assert torch.equal(loss, good)
    a, b = S.softmax_loss_backward(h, w, y, lse, one)
    assert torch.equal(a, dh) and torch.equal(b, dw)
    # others that are not finite keep to themselves
    h[[1, 2, 3]] = torch.tensor([math.nan, math.inf, -math.inf],
                                device="cuda")[:, None]
    loss, lse = S.softmax_loss_forward(h, w, y)
    assert loss[1:4].isnan().all() and torch.equal(loss[4:], good[4:])
    a, _ = S.softmax_loss_backward(h, w, y, lse, one)
    assert a[1:4].isnan().all() and torch.equal(a[4:], dh[4:])


@gpu
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
@pytest.mark.parametrize("ignore", [-1, -100, 0, 5])
def test_ignored_targets(kind, ignore):
    h, w, y = _inputs(150, 90, 40, torch.bfloat16)
    y[::3] = ignore
    _check(h, w, y.to(kind), ignore)
    y[:] = ignore
    _check(h, w, y.to(kind), ignore)


@gpu
def test_targets_out_of_range_give_nan_and_no_gradient():
    h, w, y = _inputs(140, 50, 24, torch.float32)
    y[3], y[100], y[7] = 50, -2, 2 ** 40
    loss, lse = S.softmax_loss_forward(h, w, y)
    assert loss.isnan().nonzero().flatten().tolist() == [3, 7, 100]
    assert lse.isfinite().all()
    dh, dw = S.softmax_loss_backward(h, w, y, lse,
                                     torch.ones(140, device="cuda"))
    good = torch.ones(140, dtype=torch.bool)
    good[[3, 7, 100]] = False
    assert (dh[~good] == 0).all()
    _, _, _, _, dh2, dw2, oh, ow = _reference(h[good], w, y[good],
                                              grad=torch.ones(()))
    _near(dh[good], dh2, oh, "dh")
    _near(dw, dw2, ow, "dw")


@gpu
def test_extreme_scores():
    """Scores far apart and far from 0 neither overflow nor vanish."""
    h, w, y = _inputs(40, 300, 16, torch.float32, spread=60.0)
    s = h.double() @ w.double().T
    assert s.abs().max() > 5000
    _check(h, w, y)
    one = torch.zeros(4, 8, device="cuda")
    one[:, 0] = torch.tensor([1e18, -1e18, 3e4, 0.0])
    t = torch.zeros(130, 8, device="cuda")
    t[:, 0] = -1e18
    t[129, 0] = -2e18
    loss, lse = S.softmax_loss_forward(one, t, torch.tensor(
        [0, 129, 0, 0], device="cuda"))
    assert lse.tolist()[:2] == pytest.approx([-1e36, 2e36], rel=1e-6)
    assert loss[1].item() == pytest.approx(0, abs=2e36 * 2 ** -22)
    assert lse[3].item() == pytest.approx(math.log(130), rel=1e-6)


@gpu
def test_rows_that_are_not_finite_stay_alone():
    h, w, y = _inputs(130, 64, 32, torch.bfloat16)
    h[5, 3] = math.nan
    h[129, 0] = math.inf
    loss, lse = S.softmax_loss_forward(h, w, y)
    good = torch.ones(130, dtype=torch.bool)
    good[[5, 129]] = False
    assert loss[~good].isnan().all()
    a, b, oa, ob = _reference(h[good], w, y[good])
    _near(loss[good], a, oa, "loss")
    _near(lse[good], b, ob, "lse")
    # cut off by their targets, they leave the table's gradient alone
    y[[5, 129]] = -1
    dh, dw = S.softmax_loss_backward(h, w, y, lse, torch.ones((),
                                                              device="cuda"))
    r = _reference(h[good], w, y[good], grad=torch.ones(()))
    _near(dh[good], r[4], r[6], "dh")
    _near(dw, r[5], r[7], "dw")
    assert (dh[~good] == 0).all()


@gpu
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd(reduction, dtype):
    h, w, y = _inputs(75, 410, 50, dtype)
    y[::4] = -1
    h.requires_grad_()
    w.requires_grad_()
    up = torch.linspace(-1, 2, 75, device="cuda") if reduction == "none" \
        else torch.tensor(1.7, device="cuda")
    loss = S.softmax_loss(h, w, y, reduction=reduction)
    loss.backward(up)
    kept = int((y >= 0).sum())
    g = up if reduction != "mean" else up / kept
    each, _, off, _, dh, dw, oh, ow = _reference(h.detach(), w.detach(), y,
                                                 grad=g)
    if reduction == "none":
        _near(loss.detach(), each, off, "loss")
    else:
        f = 1 if reduction == "sum" else 1 / kept
        _near(loss.detach(), each.sum() * f,
              off.sum() * f + 2 * U * each.sum() * f, "loss")
    _near(h.grad, dh, oh + 4 * U * dh.abs(), "dh")
    _near(w.grad, dw, ow + 4 * U * dw.abs(), "dw")


@gpu
def test_gradient_against_differences():
    """(L(h + e u) - L(h - e u)) / 2e against <dh, u>, and the same for w."""
    h, w, y = _inputs(20, 60, 12, torch.float32, spread=1.0)
    e = 2.0 ** -6
    loss, lse = S.softmax_loss_forward(h, w, y)
    dh, dw = S.softmax_loss_backward(h, w, y, lse,
                                     torch.ones((), device="cuda"))
    g = torch.Generator().manual_seed(3)
    for which in ("h", "w"):
        u = torch.randn(h.shape if which == "h" else w.shape,
                        generator=g).cuda()
        both = []
        for sign in (1, -1):
            a = h + sign * e * u if which == "h" else h
            b = w + sign * e * u if which == "w" else w
            both.append(S.softmax_loss_forward(a, b, y)[0].double().sum())
        got = (both[0] - both[1]) / (2 * e)
        want = ((dh if which == "h" else dw).double() * u.double()).sum()
        # along u, the scores move by t and the third derivative of their
        # log-sum-exp is t's third central moment under the softmax.  For
        # numbers within a range R that is at most R^3 max_q q (1-q) |1-2q|
        # = R^3 / (6 sqrt 3): all weight on the two ends.
        t = (u @ w.T if which == "h" else h @ u.T).double()
        wide = t.amax(1) - t.amin(1)
        off = e * e / 6 * (wide ** 3).sum() / (6 * math.sqrt(3)) \
            + 20 * 64 * U * float(loss.abs().max() + 8) / e
        assert abs(got - want) < off
        assert off < 0.2 * abs(want) + 0.5


@gpu
def test_no_rows():
    h, w, y = _inputs(0, 30, 10, torch.float32)
    loss, lse = S.softmax_loss_forward(h, w, y)
    assert loss.shape == lse.shape == (0,)
    dh, dw = S.softmax_loss_backward(h, w, y, lse, torch.zeros(0).cuda())
    assert dh.shape == (0, 10) and (dw == 0).all() and dw.shape == (30, 10)
    assert S.softmax_loss(h, w, y, reduction="sum").item() == 0
    assert math.isnan(S.softmax_loss(h, w, y).item())


@gpu
def test_only_what_is_needed():
    h, w, y = _inputs(60, 200, 30, torch.bfloat16)
    loss, lse = S.softmax_loss_forward(h, w, y)
    one = torch.ones((), device="cuda")
    dh, dw = S.softmax_loss_backward(h, w, y, lse, one)
    a, none = S.softmax_loss_backward(h, w, y, lse, one, need_w=False)
    assert none is None and torch.equal(a, dh)
    none, b = S.softmax_loss_backward(h, w, y, lse, one, need_h=False)
    assert none is None and torch.equal(b, dw)
    assert S.softmax_loss_backward(h, w, y, lse, one, need_h=False,
                                   need_w=False) == (None, None)
    w2 = w.clone().requires_grad_()
    S.softmax_loss(h, w2, y, reduction="sum").backward()
    assert torch.equal(w2.grad, dw)


@gpu
def test_the_same_on_every_run_and_on_another_stream():
    h, w, y = _inputs(333, 2500, 120, torch.bfloat16)
    one = torch.ones((), device="cuda")

    def once():
        loss, lse = S.softmax_loss_forward(h, w, y)
        return (loss, lse, *S.softmax_loss_backward(h, w, y, lse, one))
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, once()):
        assert torch.equal(a, b) and torch.equal(a, c)


@gpu
def test_captured_step():
    """A step in a graph gives the eager step's result on every replay, with
    new inputs and eager work between."""
    h, w, y = _inputs(100, 900, 72, torch.bfloat16)
    one = torch.ones((), device="cuda")

    def once(a, b, t):
        loss, lse = S.softmax_loss_forward(a, b, t)
        return (loss, *S.softmax_loss_backward(a, b, t, lse, one))
    sh, sw, sy = h.clone(), w.clone(), y.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once(sh, sw, sy)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, once(sh, sw, sy)))
    for k in range(4):
        h, w, y = _inputs(100, 900, 72, torch.bfloat16, seed=10 + k)
        sh.copy_(h), sw.copy_(w), sy.copy_(y)
        for graph, out in graphs:
            graph.replay()
        want = once(h, w, y)
        torch.cuda.synchronize()
        for graph, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [88, 350])
def test_captured_without_a_call_before(d, dtype):
    h, w, y = _inputs(45, 333, d, dtype)
    one = torch.ones((), device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, lse = S.softmax_loss_forward(h, w, y)
        dh, dw = S.softmax_loss_backward(h, w, y, lse, one)
    graph.replay()
    loss2, lse2 = S.softmax_loss_forward(h, w, y)
    dh2, dw2 = S.softmax_loss_backward(h, w, y, lse2, one)
    torch.cuda.synchronize()
    for a, b in ((loss, loss2), (lse, lse2), (dh, dh2), (dw, dw2)):
        assert torch.equal(a, b)


@gpu
def test_two_steps_before_the_first_is_read():
    """Calls that are queued behind each other do not share workspaces."""
    first = _inputs(300, 4000, 64, torch.bfloat16, seed=1)
    second = _inputs(200, 3000, 200, torch.float32, seed=2)
    one = torch.ones((), device="cuda")
    out = []
    for h, w, y in (first, second, first):
        loss, lse = S.softmax_loss_forward(h, w, y)
        out.append((loss, *S.softmax_loss_backward(h, w, y, lse, one)))
    for a, b in zip(out[0], out[2]):
        assert torch.equal(a, b)
    _check(*second)


@gpu
def test_table_past_32_bits():
    """A table of more than 2^32 bytes, with targets at its end."""
    v, d = 7_200_000, 320
    w = torch.empty(v, d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for a in range(0, v, 900_000):
        w[a:a + 900_000] = torch.randn(900_000, d, generator=g,
                                       device="cuda") * 0.2
    h = torch.randn(3, d, generator=g, device="cuda").to(torch.bfloat16)
    y = torch.tensor([v - 1, 0, v - 2], device="cuda")
    loss, lse = S.softmax_loss_forward(h, w, y)
    parts = [torch.logsumexp(h.double() @ w[a:a + 450_000].double().T, 1)
             for a in range(0, v, 450_000)]
    want = torch.logsumexp(torch.stack(parts), 0)
    right = (h.double() * w[y].double()).sum(1)
    # sums of v / 8 terms at most: see _reference
    off = (v / 8 + 64) * U + 2 * (d + 2) * U * float(
        (h.abs().double() @ w[-1000:].abs().double().T).max()) * 2 + 1e-5
    assert ((lse - want).abs() < off).all()
    assert ((loss - (want - right)).abs() < 2 * off).all()
    # no error of a wrapped offset is that small
    assert off < 0.1


def test_refusals():
    h, w = torch.zeros(4, 8), torch.zeros(10, 8)
    y = torch.zeros(4, dtype=torch.long)
    for bad, error in (
            (([1.0], w, y), TypeError), ((h, w, [0]), TypeError),
            ((h[0], w, y), ValueError), ((h, w[0], y), ValueError),
            ((h, w, y[:, None]), ValueError),
            ((h, w[:, :7], y), ValueError), ((h[:3], w, y), ValueError),
            ((h, w[:0], y), ValueError), ((h[:, :0], w[:, :0], y), ValueError),
            ((torch.zeros(4, 2 ** 20 + 1), torch.zeros(1, 2 ** 20 + 1), y),
             ValueError),
            ((h.half(), w.half(), y), TypeError),
            ((h.double(), w.double(), y), TypeError),
            ((h, w.bfloat16(), y), TypeError),
            ((h, w, y.to(torch.int16)), TypeError),
            ((h, w, y.float()), TypeError), ((h, w, y), RuntimeError)):
        with pytest.raises(error):
            S.softmax_loss(*bad)
        with pytest.raises(error):
            S.softmax_loss_forward(*bad)
    with pytest.raises(ValueError):
        S.softmax_loss(h, w, y, reduction="avg")
    with pytest.raises(RuntimeError):
        S.softmax_loss_backward(h, w, y, torch.zeros(4), torch.zeros(4))


@gpu
def test_refusals_of_the_backward():
    h, w, y = _inputs(4, 10, 8, torch.float32)
    one, lse = torch.ones((), device="cuda"), torch.zeros(4, device="cuda")
    for bad in ((lse[:3], one), (lse.double(), one), (lse, lse[:3]),
                (lse, lse[:, None]), (lse, one.half())):
        with pytest.raises(ValueError):
            S.softmax_loss_backward(h, w, y, *bad)
    with pytest.raises(TypeError):
        S.softmax_loss_backward(h, w, y, lse, 1.0)
    with pytest.raises(RuntimeError):
        S.softmax_loss_backward(h, w, y, lse.cpu(), one)
    with pytest.raises(RuntimeError):
        S.softmax_loss(h, w.cpu(), y)


@gpu
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_loss_may_be_changed_in_place(reduction):
    """loss /= 4 before backward(), as when gradients are accumulated: a power
    of two, so that the gradients are a quarter to the last bit."""
    h, w, y = _inputs(50, 400, 24, torch.float32)
    grads = []
    for change in (False, True):
        a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
        loss = S.softmax_loss(a, b, y, reduction=reduction)
        if change:
            loss /= 4
        loss.sum().backward()
        grads.append((a.grad, b.grad))
    for one, quarter in zip(*grads):
        assert torch.equal(one / 4, quarter)


@gpu
def test_gradients_are_not_captured(monkeypatch):
    h, w, y = _inputs(20, 100, 24, torch.float32)
    a = h.clone().requires_grad_()
    loss = S.softmax_loss(a, w, y)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            S.softmax_loss(a, w, y)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            loss.backward(retain_graph=True)
        assert torch.equal(S.softmax_loss(h, w, y), loss.detach())
    loss.backward()
    assert a.grad is not None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        out = S.softmax_loss(a, w, y)
    graph.replay()
    assert torch.equal(out, loss.detach())


@gpu
def test_two_threads_with_their_own_streams():
    """Calls that run at the same time keep to their own workspaces."""
    import threading
    cases = [_inputs(300, 4000, 64, torch.bfloat16, seed=1),
             _inputs(250, 50_000, 100, torch.float32, seed=2)]
    one = torch.ones((), device="cuda")

    def once(h, w, y):
        loss, lse = S.softmax_loss_forward(h, w, y, gradient=True)
        return (loss, *S.softmax_loss_backward(h, w, y, lse, one))
    want = [once(*case) for case in cases]
    torch.cuda.synchronize()
    bad = []

    def work(case, ref):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                for a, b in zip(once(*case), ref):
                    if not torch.equal(a, b):
                        bad.append(len(case[0]))
    threads = [threading.Thread(target=work, args=pair)
               for pair in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@gpu
@pytest.mark.parametrize("n,v,d", [(300, 40_000, 100), (40, 300, 700)])
def test_captured_float32(n, v, d):
    """Parts of bfloat16 and small tiles, with new inputs on every replay."""
    h, w, y = _inputs(n, v, d, torch.float32)
    one = torch.ones((), device="cuda")

    def once(a, b, t):
        loss, lse = S.softmax_loss_forward(a, b, t, gradient=True)
        return (loss, *S.softmax_loss_backward(a, b, t, lse, one))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once(h, w, y)
    for k in range(4):
        a, b, t = _inputs(n, v, d, torch.float32, seed=20 + k)
        h.copy_(a), w.copy_(b), y.copy_(t)
        graph.replay()
        want = once(a, b, t)
        torch.cuda.synchronize()
        for x, z in zip(out, want):
            assert torch.equal(x, z)
