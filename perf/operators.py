"""The operators over the whole vocabulary, and what they are measured on.

  loss      softmax cross entropy of N rows against a table of V word rows,
            and the log of the softmax's sum
  grad      the same with the mean's gradients to the rows and to the table
  rows      rows to 8-bit floats with a power-of-two scale for each block of
            128 columns, and back to the values they stand for
  scores    product of query rows, held like that, with such a table: cosine
            scores of every query against every word

``run`` computes them in plain torch operations, or with ``own`` by the
framework's kernels.  Tables lie as the framework keeps them: rows padded with
zeros to a multiple of 64 columns.
"""
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one context scored against the headline vocabulary: bound by the
        # table's bytes
        {"name": "loss 1 of 1M x 300", "op": "loss", "n": 1,
         "v": 1_000_000, "d": 300, "dtype": "bfloat16", "ignored": 0.0},
        # held-out pairs of a small corpus with the default vector size
        {"name": "loss 2000 of 3613 x 100 f32", "op": "loss", "n": 2000,
         "v": 3613, "d": 100, "dtype": "float32", "ignored": 0.05},
        # held-out pairs of the headline vocabulary
        {"name": "loss 4096 of 1M x 300", "op": "loss", "n": 4096,
         "v": 1_000_000, "d": 300, "dtype": "bfloat16", "ignored": 0.0},
        # one small step: latency counts
        {"name": "grad 256 of 10k x 128", "op": "grad", "n": 256,
         "v": 10_000, "d": 128, "dtype": "bfloat16", "ignored": 0.0},
        # a step on a small corpus, in 32 bits, some pairs cut off
        {"name": "grad 1000 of 3613 x 100 f32", "op": "grad", "n": 1000,
         "v": 3613, "d": 100, "dtype": "float32", "ignored": 0.05},
        # an exact step at the headline vocabulary and dimension
        {"name": "grad 4096 of 1M x 300", "op": "grad", "n": 4096,
         "v": 1_000_000, "d": 300, "dtype": "bfloat16", "ignored": 0.0},
        # a step at the high dimension, odd sizes
        {"name": "grad 2047 of 100001 x 1024", "op": "grad", "n": 2047,
         "v": 100_001, "d": 1024, "dtype": "bfloat16", "ignored": 0.02},
        # a batch of queries brought to 8 bits
        {"name": "rows 33 x 100 f32", "op": "rows", "n": 33, "d": 100,
         "dtype": "float32"},
        # the headline table brought to 8 bits
        {"name": "rows 1M x 300", "op": "rows", "n": 1_000_000, "d": 300,
         "dtype": "bfloat16"},
        # one query against the headline table
        {"name": "scores 1 of 1M x 300", "op": "scores", "n": 1,
         "v": 1_000_000, "d": 300, "dtype": "float32", "out": "float32"},
        # the batched serving size
        {"name": "scores 4096 of 200k x 300", "op": "scores", "n": 4096,
         "v": 200_000, "d": 300, "dtype": "float32", "out": "float32"},
        # an odd batch at the high dimension, scores in 16 bits
        {"name": "scores 1023 of 150001 x 1024", "op": "scores", "n": 1023,
         "v": 150_001, "d": 1024, "dtype": "bfloat16", "out": "bfloat16"},
    ]


def _log_uniform(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(("loss", "grad", "rows", "scores"))
    d = _log_uniform(rng, 16, 1024)
    case = {"op": op, "d": d, "dtype": rng.choice(("float32", "bfloat16"))}
    if op == "rows":
        return {**case, "n": _log_uniform(rng, 1, 400_000)}
    n, v = _log_uniform(rng, 1, 8192), _log_uniform(rng, 2, 500_000)
    if op == "scores":
        return {**case, "n": n, "v": min(v, 400_000_000 // n),
                "out": rng.choice(("float32", "bfloat16"))}
    # 32-bit products cost more: fewer of them
    most = 4e11 if case["dtype"] == "bfloat16" else 4e10
    return {**case, "n": n, "v": max(2, min(v, int(most / (n * d)))),
            "ignored": rng.choice((0.0, 0.1))}


def work(case):
    n, d = case["n"], case["d"]
    size = DTYPES[case["dtype"]].itemsize
    blocks = -(-d // 128)
    if case["op"] == "rows":
        # rows in, 8-bit values and scales out and in again, values out
        return {"bytes": n * (d * (size + 4) + 2 * blocks),
                "flops": 2 * n * d}
    v = case["v"]
    if case["op"] == "scores":
        return {"bytes": n * d * size + v * (d + blocks + 4)
                + n * v * DTYPES[case["out"]].itemsize,
                "flops": 2 * n * v * d}
    rows = (n + v) * d * size
    if case["op"] == "loss":
        return {"bytes": rows + 8 * n + 8 * n, "flops": 2 * n * v * d}
    # scores once, two products with their gradient
    return {"bytes": 2 * rows + 8 * n, "flops": 6 * n * v * d}


def _table(rows, d, dtype, gen, spread):
    """Rows padded with zeros as the framework keeps them, as [rows, d]."""
    stride = -(-d // 64) * 64
    t = torch.zeros(rows, stride, dtype=dtype, device="cuda")
    # words differ in length, as they do after training
    length = torch.rand(rows, 1, generator=gen, device="cuda") + 0.5
    t[:, :d] = (torch.randn(rows, d, generator=gen, device="cuda")
                * (length * spread)).to(dtype)
    return t[:, :d]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, n, d = case["op"], case["n"], case["d"]
    dtype = DTYPES[case["dtype"]]
    state = {"op": op}
    if op == "rows":
        state["x"] = _table(n, d, dtype, gen, 0.3)
        return state
    v = case["v"]
    if op == "scores":
        q = torch.randn(n, d, generator=gen, device="cuda")
        state["q"] = (q / q.norm(dim=1, keepdim=True)).to(dtype)
        w = _table(v, d, torch.bfloat16, gen, 0.3)
        state["inv_norms"] = 1.0 / w.float().norm(dim=1).clamp_min(1e-12)
        # the 8-bit table that a serving program holds: rows start at
        # multiples of 16 bytes
        values, scales = _quantize(w)
        held = torch.zeros(v, -(-d // 16) * 16, dtype=torch.uint8,
                           device="cuda")
        held[:, :d] = values.view(torch.uint8)
        state["values"] = held.view(torch.float8_e4m3fn)[:, :d]
        state["scales"] = scales.to(torch.float8_e8m0fnu)
        state["out"] = DTYPES[case["out"]]
        return state
    # logits spread by about two, as after some training
    state["h"] = _table(n, d, dtype, gen, 1.4 * d ** -0.25)
    state["w"] = _table(v, d, dtype, gen, 1.4 * d ** -0.25)
    # frequent words come first
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    y = (v ** u - 1).long().clamp_(0, v - 1)
    if case["ignored"]:
        y[torch.rand(n, generator=gen, device="cuda") < case["ignored"]] = -1
        y[0] = 0
    state["y"] = y
    return state


# -- plain forms, in 32 bits --------------------------------------------------

def _blocks(x):
    """[R, K] to [R, blocks, 128], with zeros behind the last column."""
    r, k = x.shape
    full = torch.zeros(r, -(-k // 128) * 128, dtype=x.dtype, device=x.device)
    full[:, :k] = x
    return full.view(r, -1, 128)


def _quantize(x):
    """8-bit values [R, K] and their scales, powers of two, as float32."""
    b = _blocks(x.float())
    mantissa, exponent = torch.frexp(b.abs().amax(dim=2))
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    scales = torch.ldexp(torch.ones_like(mantissa), e.clamp(-120, 120))
    values = (b / scales[:, :, None]).to(torch.float8_e4m3fn)
    return values.view(x.shape[0], -1)[:, :x.shape[1]], scales


def _dequantize(values, scales):
    return (_blocks(values.float()) * scales.float()[:, :, None]) \
        .view(values.shape[0], -1)[:, :values.shape[1]]


def _plain_scores(state):
    a = _dequantize(*_quantize(state["q"]))
    b = _dequantize(state["values"], state["scales"])
    return ((a @ b.T) * state["inv_norms"]).to(state["out"])


def _plain_loss(h, w, y):
    s = h.float() @ w.float().T
    top = s.amax(dim=1, keepdim=True)
    s = s.sub_(top).exp_()
    total = s.sum(dim=1, keepdim=True)
    lse = (top + total.log()).squeeze(1)
    kept = y >= 0
    right = (h.float() * w.float()[y.clamp_min(0)]).sum(dim=1)
    loss = torch.where(kept, lse - right, torch.zeros_like(lse))
    return loss, lse, s, total, kept


def _plain_grad(h, w, y):
    loss, _, s, total, kept = _plain_loss(h, w, y)
    each = kept.float() / kept.sum()
    c = s.mul_(each[:, None] / total)
    c[torch.arange(len(y), device=y.device), y.clamp_min(0)] -= each
    return ((loss * each).sum(), (c @ w.float()).to(h.dtype),
            (c.T @ h.float()).to(w.dtype))


def run(state):
    op = state["op"]
    if own:
        from glint_word2vec_amd.ops import fp8, softmax
        if op == "loss":
            return softmax.softmax_loss_forward(state["h"], state["w"],
                                                state["y"])
        if op == "grad":
            h = state["h"].detach().requires_grad_()
            w = state["w"].detach().requires_grad_()
            loss = softmax.softmax_loss(h, w, state["y"])
            return (loss.detach(), *torch.autograd.grad(loss, (h, w)))
        if op == "rows":
            return fp8.dequantize_rows(fp8.quantize_rows(state["x"]),
                                       dtype=torch.bfloat16)
        return fp8.matmul_rows(
            state["q"], fp8.Fp8Rows(state["values"], state["scales"]),
            col_scale=state["inv_norms"], out_dtype=state["out"])
    if op == "loss":
        return _plain_loss(state["h"], state["w"], state["y"])[:2]
    if op == "grad":
        return _plain_grad(state["h"], state["w"], state["y"])
    if op == "rows":
        # three bits behind the point and a power of two: 16 bits hold it
        return _dequantize(*_quantize(state["x"])).to(torch.bfloat16)
    return _plain_scores(state)


# -- the definitions in 64 bits -----------------------------------------------

def _held(x):
    """What rows stand for once they are held in 8 bits: the nearest number
    of 1 + 3 binary digits (ties to even) from 2^-9 up, in units of the
    smallest power of two that keeps the block within 448."""
    x = x.double()
    out = torch.zeros_like(x)
    for k in range(0, x.shape[1], 128):
        b = x[:, k:k + 128]
        most = b.abs().amax(dim=1, keepdim=True)
        e = torch.ceil(torch.log2(most / 448)).clamp(-120, 120)
        unit = torch.exp2(e)
        u = b / unit
        step = torch.exp2(
            torch.floor(torch.log2(u.abs())).clamp_min(-6) - 3)
        out[:, k:k + 128] = torch.round(u / step) * step * unit
    return out


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "rows":
        return _held(state["x"])
    if op == "scores":
        value = state["values"].double()
        for k, s in enumerate(state["scales"].double().unbind(1)):
            value[:, 128 * k:128 * k + 128] *= s[:, None]
        return _held(state["q"]) @ value.T * state["inv_norms"].double()
    h, w, y = state["h"].double(), state["w"].double(), state["y"]
    n, v = len(h), len(w)
    step = max(1, 2 ** 28 // n)
    lse = torch.full((n,), -torch.inf, dtype=torch.float64, device="cuda")
    for a in range(0, v, step):
        lse = torch.logaddexp(lse, torch.logsumexp(h @ w[a:a + step].T, 1))
    kept = y >= 0
    loss = torch.zeros_like(lse)
    loss[kept] = lse[kept] - (h[kept] * w[y[kept]]).sum(1)
    if op == "loss":
        return loss, lse
    h, lse, y = h[kept], lse[kept], y[kept]
    dh, dw = torch.zeros_like(state["h"], dtype=torch.float64), \
        torch.zeros_like(w)
    part = torch.zeros_like(h)
    for a in range(0, v, step):
        p = torch.exp(h @ w[a:a + step].T - lse[:, None])
        here = ((y >= a) & (y < a + step)).nonzero().squeeze(1)
        p[here, y[here] - a] -= 1
        part += p @ w[a:a + step]
        dw[a:a + step] = p.T @ h
    dh[kept] = part / len(y)
    return loss.sum() / len(y), dh, dw / len(y)
