"""Softmax cross entropy over the whole vocabulary, by hand-written kernels.

Negative sampling trains on a handful of sampled words because the softmax
over the vocabulary was out of reach; on this hardware it is one matrix
product per direction.  For rows ``h`` [N, D], a table ``w`` [V, D] and target
words ``y`` [N]

    lse_n  = log sum_v exp <h_n, w_v>       loss_n = lse_n - <h_n, w_y(n)>

The scores [N, V] are never kept: the loss is one pass over the table with a
running maximum and sum, and the gradient takes the vocabulary in pieces.
Products and sums are held in 32 bits; for bfloat16 tables the gradient's
coefficients are rounded to bfloat16 before the products with the rows.

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
    if max(h.shape[0], w.shape[0]) > 2 ** 31 - 1024 or w.shape[1] > 1 << 24:
        raise ValueError("at most 2^31 - 1024 rows of 2^24 columns")
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


def _forward(h, w, targets, ignore_index, reduce: int):
    """(loss [N], lse [N], [reduced loss, factor] or None)."""
    _check(h, w, targets)
    h, w, targets = _rows(h.detach()), _rows(w.detach()), targets.contiguous()
    n, d = h.shape
    v = w.shape[0]
    loss = torch.empty(n, dtype=torch.float32, device=h.device)
    lse = torch.empty_like(loss)
    reduced = torch.empty(2, dtype=torch.float32, device=h.device) \
        if reduce else None
    size, dp = h.element_size(), _ceil(d, 64) * 64
    packed_h = packed_w = None
    piece = v
    if not _aligned(h):
        packed_h = torch.empty(n * dp, dtype=h.dtype, device=h.device)
    # (the kernel for few rows streams any table)
    if not _aligned(w) and not (n <= 16 and d * size <= 4096):
        piece = max(256, _PACKED_BYTES // (dp * size) // 256 * 256)
        packed_w = torch.empty(min(piece, v) * dp, dtype=w.dtype,
                               device=w.device)
    # a maximum and a sum of every row for each part of the vocabulary
    parts = max(_ceil(v, piece), min(_ceil(v, 64),
                                     _PARTS // max(1, _ceil(n, 128))))
    part = torch.empty(parts * n * 2, dtype=torch.float32, device=h.device)
    _native().softmax_loss(
        h.data_ptr(), h.stride(0), n, w.data_ptr(), w.stride(0), v, d,
        int(h.dtype == torch.bfloat16), targets.data_ptr(),
        int(targets.dtype == torch.int64), int(ignore_index),
        part.data_ptr(), parts * n,
        0 if packed_h is None else packed_h.data_ptr(),
        0 if packed_w is None else packed_w.data_ptr(), piece,
        loss.data_ptr(), lse.data_ptr(), reduce,
        0 if reduced is None else reduced.data_ptr(), *_place(h.device))
    return loss, lse, reduced


def _backward(h, w, targets, lse, grad, weight, ignore_index, need_h, need_w):
    h, w, targets = _rows(h.detach()), _rows(w.detach()), targets.contiguous()
    n, d = h.shape
    v = w.shape[0]
    dh = torch.empty((n, d), dtype=h.dtype, device=h.device) \
        if need_h else None
    if n == 0 or not (need_h or need_w):
        return dh, (torch.zeros((v, d), dtype=w.dtype, device=w.device)
                    if need_w else None)
    dw = torch.empty((v, d), dtype=w.dtype, device=w.device) \
        if need_w else None
    size = h.element_size()
    rows = _ceil(n, 32) * 32
    packed = torch.empty(rows * _ceil(d, 64) * 64, dtype=h.dtype,
                         device=h.device)
    # equal pieces of the vocabulary, in whole tiles
    pieces = _ceil(v, max(256, _COEF_BYTES // (rows * size)))
    width = _ceil(_ceil(v, pieces), 256) * 256
    coef = torch.empty(rows * width, dtype=h.dtype, device=h.device)
    packed_w = None if _aligned(w) else \
        torch.empty(width * _ceil(d, 64) * 64, dtype=w.dtype, device=w.device)
    ldp = _ceil(d, 4) * 4
    # parts of the long axis where a product's result has few tiles
    splits, splits_w = _native().softmax_plan(n, min(v, width), d,
                                              int(size == 2))
    splits_w = splits_w if need_w else 1
    part = torch.empty(splits * n * ldp if need_h else 0,
                       dtype=torch.float32, device=h.device)
    part_w = torch.empty(splits_w * width * ldp if splits_w > 1 else 0,
                         dtype=torch.float32, device=h.device)
    _native().softmax_grad(
        h.data_ptr(), h.stride(0), n, w.data_ptr(), w.stride(0), v, d,
        int(h.dtype == torch.bfloat16), targets.data_ptr(),
        int(targets.dtype == torch.int64), int(ignore_index), lse.data_ptr(),
        grad.data_ptr(), int(grad.dim() > 0),
        0 if weight is None else weight.data_ptr(), packed.data_ptr(),
        0 if packed_w is None else packed_w.data_ptr(), width,
        coef.data_ptr(), splits, part.data_ptr() if need_h else 0, splits_w,
        part_w.data_ptr() if splits_w > 1 else 0, ldp,
        0 if dh is None else dh.data_ptr(),
        0 if dw is None else dw.data_ptr(), *_place(h.device))
    return dh, dw


class _SoftmaxLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, targets, reduce, ignore_index):
        loss, lse, reduced = _forward(h, w, targets, ignore_index, reduce)
        ctx.save_for_backward(h, w, targets, lse,
                              None if reduced is None else reduced[1])
        ctx.ignore_index = ignore_index
        return loss if reduced is None else reduced[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        h, w, targets, lse, weight = ctx.saved_tensors
        dh, dw = _backward(h, w, targets, lse,
                           grad.to(torch.float32).contiguous(), weight,
                           ctx.ignore_index, *ctx.needs_input_grad[:2])
        return dh, dw, None, None, None


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
    loss is NaN, and it gives no gradient.  Rows whose scores are not finite
    give NaN."""
    if reduction not in _REDUCE:
        raise ValueError(f"reduction must be one of {sorted(_REDUCE)}, got "
                         f"{reduction!r}")
    return _SoftmaxLoss.apply(h, w, targets, _REDUCE[reduction],
                              int(ignore_index))


def softmax_loss_forward(h: torch.Tensor, w: torch.Tensor,
                         targets: torch.Tensor, ignore_index: int = -1
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The loss and the log of the softmax's sum, both float32 [N], without
    autograd (evaluation, or a captured step together with
    softmax_loss_backward).  Targets as for softmax_loss."""
    return _forward(h, w, targets, ignore_index, 0)[:2]


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
    return _backward(h, w, targets, lse.detach().contiguous(),
                     grad.detach().contiguous(), None, ignore_index, need_h,
                     need_w)
