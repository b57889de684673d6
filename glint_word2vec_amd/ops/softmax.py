"""Softmax cross entropy over the whole vocabulary, by hand-written kernels.

Negative sampling trains on a handful of sampled words because the softmax
over the vocabulary was out of reach; on this hardware it is one matrix
product per direction.  For rows ``h`` [N, D], a table ``w`` [V, D] and target
words ``y`` [N]

    lse_n  = log sum_v exp <h_n, w_v>       loss_n = lse_n - <h_n, w_y(n)>

The scores [N, V] are never kept: the loss is one pass over the table with a
running maximum and sum, and the gradient takes the vocabulary in pieces.
Sums are held in 32 bits; for bfloat16 tables the gradient's coefficients are
rounded to bfloat16 before the products with the rows.  That adds 2 to 5% to
the error that the gradient's own rounding to bfloat16 makes;
softmax_loss(h.float(), w.float(), targets) gives gradients without it, in up to
five times the time.  float32 products of many samples are made of three
bfloat16 parts of each number, which loses no more than float32's own rounding.

Every function runs on the current stream of the tensors' device, allocates
its workspace from torch's allocator for the one call, and does not
synchronise.  Results are the same on every run: there are no atomics.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

# Pieces of the vocabulary are as wide as keeps their coefficients within
# this, and packed copies of unaligned tables within that.
_COEF_BYTES = 1 << 30
_PACKED_BYTES = 256 << 20
_PARTS = 4096


def _native():
    try:
        from .. import _vocab_native
        return _vocab_native
    except ImportError as e:
        raise RuntimeError(
            "glint_word2vec_amd._vocab_native is not built but a GPU path was "
            "requested. Build it in-tree with `python setup.py build_ext "
            "--inplace` (hipcc, gfx950). Refusing to fall back to eager."
        ) from e


def _place(device: torch.device) -> Tuple[int, int]:
    """Device and stream that a call is launched on."""
    return device.index, torch.cuda.current_stream(device).cuda_stream


def _ceil(a: int, b: int) -> int:
    return -(-a // b)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows whose elements are neighbours; any distance between rows."""
    if t.shape[0] <= 1 or t.shape[1] <= 1:
        return t.contiguous()
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] \
        else t.contiguous()


def _check(h, w, targets) -> None:
    for name, t in (("h", h), ("w", w), ("targets", targets)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if h.dim() != 2 or w.dim() != 2 or targets.dim() != 1:
        raise ValueError(
            "expected h [N, D], w [V, D] and targets [N], got "
            f"{list(h.shape)}, {list(w.shape)}, {list(targets.shape)}")
    if h.shape[1] != w.shape[1]:
        raise ValueError(f"h has {h.shape[1]} columns, w has {w.shape[1]}")
    if h.shape[0] != targets.shape[0]:
        raise ValueError(f"{h.shape[0]} rows but {targets.shape[0]} targets")
    if w.shape[0] < 1 or w.shape[1] < 1:
        raise ValueError("the vocabulary needs a word and a column")
    if h.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported dtype {h.dtype}: float32 or bfloat16")
    if w.dtype != h.dtype:
        raise TypeError(f"h is {h.dtype} but w is {w.dtype}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"targets must be int32 or int64, got {targets.dtype}")
    if max(h.shape[0], w.shape[0]) > 2 ** 31 - 1024 or w.shape[1] > 1 << 20:
        raise ValueError("at most 2^31 - 1024 rows of 2^20 columns")
    if not (h.is_cuda and w.is_cuda and targets.is_cuda):
        raise RuntimeError("the softmax kernels run on the GPU: move h, w and "
                           "targets there")
    if not (h.device == w.device == targets.device):
        raise RuntimeError("h, w and targets are on different devices: "
                           f"{h.device}, {w.device}, {targets.device}")


def _aligned(t: torch.Tensor) -> bool:
    """Whether the kernels read rows as they lie: they start at multiples of
    16 bytes, less than 2^23 bytes apart."""
    step = t.stride(0) * t.element_size()
    return t.data_ptr() % 16 == 0 and step % 16 == 0 and step < 1 << 23


# How the kernels take the numbers, and bytes of one: float32, bfloat16, and
# float32 in three parts of bfloat16 (see kSplit in the kernels' source).
_FLOAT, _BF16, _SPLIT = 0, 1, 3
_BYTES = {_FLOAT: 4, _BF16: 2, _SPLIT: 6}
# float32 goes in parts from so many samples and products on; see _kind
_SPLIT_LOSS = 384, 1 << 31
_SPLIT_GRAD = 192, 1 << 30
_SPLIT_COEF_BYTES = 256 << 20


def _kind(h: torch.Tensor, v: int, grad: bool) -> int:
    """How this call takes its numbers: with `grad` for a gradient and the lse
    that it starts from.  A coefficient exp(s - lse) is exact to a part of the
    score's own error, as its score and those in lse were rounded alike; an lse
    of the other form costs that (285 x 95 x 588: 1.6e-6 instead of 5e-7 of
    the gradient).  In parts the products run faster, but
    the table is written once more and the coefficients take half as much
    again.  Times in float32 and in parts (us):
      loss, d = 200: 512 x 30000 71 and 63, 4096 x 30000 438 and 300;
        256 x 200000 202 and 252, 1024 x 4000 28 and 37
      loss with its gradient, d = 300: 3000 x 3000 357 and 232, 8000 x 1000
        305 and 215; 1000 x 1000 85 and 115, 300 x 3000 82 and 116
      gradient, d = 64: 512 x 200000 438 and 556, whose coefficients are past
        the cache"""
    if h.dtype == torch.bfloat16:
        return _BF16
    n, d = h.shape
    rows, products = _SPLIT_GRAD if grad else _SPLIT_LOSS
    if n < rows or n * v * d < products:
        return _FLOAT
    if grad and d < 96 and n * v * _BYTES[_SPLIT] > _SPLIT_COEF_BYTES:
        return _FLOAT
    return _SPLIT


def _workspace(device, *sizes: int) -> Tuple[torch.Tensor, list]:
    """One allocation for parts of these many bytes, and where they start
    (0 for a part of none); hold the tensor until the launches are made."""
    starts, total = [], 0
    for size in sizes:
        starts.append(total)
        total += _ceil(size, 256) * 256
    held = torch.empty(total, dtype=torch.uint8, device=device)
    base = held.data_ptr()
    return held, [base + at if size else 0
                  for at, size in zip(starts, sizes)]


def _forward(h, w, targets, ignore_index, reduce: int, grad: bool):
    """(loss [N], lse [N], reduced loss or None, its factor or None)."""
    _check(h, w, targets)
    h, w, targets = _rows(h), _rows(w), targets.contiguous()
    (n, d), v, device = h.shape, w.shape[0], h.device
    loss = torch.empty(n, dtype=torch.float32, device=device)
    lse = torch.empty_like(loss)
    result = factor = None
    if reduce:      # two tensors: the result may be changed in place
        result = torch.empty((), dtype=torch.float32, device=device)
        factor = torch.empty_like(result)
    size = h.element_size()
    kind = _kind(h, v, grad)
    row = _ceil(d, 64) * 64 * _BYTES[kind]    # of a packed row
    piece = v
    # (the kernel for few rows streams any table)
    pack_w = kind == _SPLIT or not _aligned(w) and not (
        n <= 16 and d * size <= 4096)
    if pack_w:
        piece = max(256, _PACKED_BYTES // row // 256 * 256)
    # a maximum and a sum of every row for each part of the vocabulary
    parts = max(_ceil(v, piece), min(_ceil(v, 64),
                                     _PARTS // max(1, _ceil(n, 128))))
    held, (part, packed_h, packed_w) = _workspace(
        device, parts * n * 8,
        0 if kind != _SPLIT and _aligned(h) else n * row,
        min(piece, v) * row if pack_w else 0)
    _native().softmax_loss(
        h.data_ptr(), h.stride(0), n, w.data_ptr(), w.stride(0), v, d,
        kind, targets.data_ptr(),
        int(targets.dtype == torch.int64), ignore_index, part, parts * n,
        packed_h, packed_w, piece, loss.data_ptr(), lse.data_ptr(), reduce,
        0 if result is None else result.data_ptr(),
        0 if factor is None else factor.data_ptr(), *_place(device))
    return loss, lse, result, factor


def _backward(h, w, targets, lse, grad, factor, ignore_index, need_h, need_w):
    h, w, targets = _rows(h), _rows(w), targets.contiguous()
    (n, d), v, device = h.shape, w.shape[0], h.device
    dh = torch.empty((n, d), dtype=h.dtype, device=device) \
        if need_h else None
    if n == 0 or not (need_h or need_w):
        return dh, (torch.zeros((v, d), dtype=w.dtype, device=device)
                    if need_w else None)
    dw = torch.empty((v, d), dtype=w.dtype, device=device) \
        if need_w else None
    native = _native()
    kind = _kind(h, v, True)
    size = _BYTES[kind]
    rows, row = _ceil(n, 32) * 32, _ceil(d, 64) * 64 * size
    # equal pieces of the vocabulary, in whole tiles
    most = rows * size if kind != _SPLIT else max(rows * size, row)
    pieces = _ceil(v, max(256, _COEF_BYTES // most))
    width = _ceil(_ceil(v, pieces), 256) * 256
    # parts of the long axis where a product's result has few tiles
    splits, splits_w = native.softmax_plan(n, min(v, width), d, kind)
    ldp = _ceil(d, 4) * 4
    held, (packed, packed_w, coef, part, part_w) = _workspace(
        device, rows * row,
        0 if kind != _SPLIT and _aligned(w) else width * row,
        rows * width * size, splits * n * ldp * 4 if need_h else 0,
        splits_w * width * ldp * 4 if need_w and splits_w > 1 else 0)
    native.softmax_grad(
        h.data_ptr(), h.stride(0), n, w.data_ptr(), w.stride(0), v, d,
        kind, targets.data_ptr(),
        int(targets.dtype == torch.int64), ignore_index, lse.data_ptr(),
        grad.data_ptr(), int(grad.dim() > 0),
        0 if factor is None else factor.data_ptr(), packed, packed_w, width,
        coef, splits, part, splits_w, part_w, ldp,
        0 if dh is None else dh.data_ptr(),
        0 if dw is None else dw.data_ptr(), *_place(device))
    return dh, dw


def _refuse_capture() -> None:
    # Leaves keep one gradient node per eager graph that lives, bound to that
    # graph's stream; a captured backward that meets one ends the process.
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(
            "softmax_loss with gradients cannot be captured: capture "
            "softmax_loss_forward and softmax_loss_backward")


class _SoftmaxLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, targets, reduce, ignore_index, grad):
        loss, lse, result, factor = _forward(h, w, targets, ignore_index,
                                             reduce, grad)
        ctx.ignore_index = ignore_index
        ctx.save_for_backward(h, w, targets, lse,
                              *(() if factor is None else (factor,)))
        return loss if result is None else result

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _refuse_capture()
        h, w, targets, lse, *factor = ctx.saved_tensors
        if grad.dtype != torch.float32 or not grad.is_contiguous():
            grad = grad.to(torch.float32).contiguous()
        return (*_backward(h, w, targets, lse, grad,
                           factor[0] if factor else None, ctx.ignore_index,
                           *ctx.needs_input_grad[:2]), None, None, None, None)


_REDUCE = {"none": 0, "sum": 1, "mean": 2}


def softmax_loss(h: torch.Tensor, w: torch.Tensor, targets: torch.Tensor,
                 reduction: str = "mean",
                 ignore_index: int = -1) -> torch.Tensor:
    """Cross entropy of rows ``h`` [N, D] against the table ``w`` [V, D] with
    target words ``targets`` [N] (int32 or int64), differentiable in ``h`` and
    ``w`` (float32 or bfloat16, the same for both).

    ``reduction``: "mean" over the targets that count, "sum", or "none" for
    the loss [N].  Losses are float32.  Targets equal to ``ignore_index``
    count nothing and give no gradient (the mean of none is NaN).  Any other
    target outside [0, V) cannot be refused without waiting for the GPU: its
    loss is NaN, and it gives no gradient.  A score of NaN or +inf makes its row
    NaN, and so does one of -inf for every word; otherwise a score of -inf is a
    probability of 0.  A score past float32's range counts as infinite, or, where
    float32 goes in parts, as NaN.  A call that needs gradients is refused while
    a graph is being captured: softmax_loss_forward and softmax_loss_backward
    can be."""
    if reduction not in _REDUCE:
        raise ValueError(f"reduction must be one of {sorted(_REDUCE)}, got "
                         f"{reduction!r}")
    grad = torch.is_grad_enabled() and any(
        getattr(t, "requires_grad", False) for t in (h, w))
    if grad:
        _refuse_capture()
    return _SoftmaxLoss.apply(h, w, targets, _REDUCE[reduction],
                              int(ignore_index), grad)


def softmax_loss_forward(h: torch.Tensor, w: torch.Tensor,
                         targets: torch.Tensor, ignore_index: int = -1,
                         gradient: bool = False
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The loss and the log of the softmax's sum, both float32 [N], without
    autograd (evaluation, or a captured step together with
    softmax_loss_backward).  Targets as for softmax_loss.  With ``gradient``
    scores are rounded as softmax_loss_backward rounds them: its gradient is
    then the most exact."""
    with torch.no_grad():
        return _forward(h, w, targets, int(ignore_index), 0,
                        bool(gradient))[:2]


def softmax_loss_backward(h: torch.Tensor, w: torch.Tensor,
                          targets: torch.Tensor, lse: torch.Tensor,
                          grad: torch.Tensor, ignore_index: int = -1,
                          need_h: bool = True, need_w: bool = True
                          ) -> Tuple[Optional[torch.Tensor],
                                     Optional[torch.Tensor]]:
    """Gradients (to ``h``, to ``w``) of sum_n grad_n loss_n, in the tables'
    dtype.  ``lse`` is what softmax_loss_forward gave; ``grad`` is float32
    [N], or one number [] for all rows."""
    _check(h, w, targets)
    n = h.shape[0]
    for name, t, shapes in (("lse", lse, ([n],)), ("grad", grad, ([n], []))):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
        if t.dtype != torch.float32 or list(t.shape) not in shapes:
            raise ValueError(f"{name} must be float32 of shape "
                             f"{' or '.join(map(str, shapes))}, got {t.dtype} "
                             f"{list(t.shape)}")
        if t.device != h.device:
            raise RuntimeError(f"{name} is on {t.device}, h on {h.device}")
    with torch.no_grad():
        return _backward(h, w, targets, lse.contiguous(), grad.contiguous(),
                         None, int(ignore_index), need_h, need_w)
