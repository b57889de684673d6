"""Rows in 8-bit floats with a scale for each block of 128 columns, and their
matrix product, by hand-written kernels.

A row's block of up to 128 columns is held as e4m3 values times one power of
two, the smallest that keeps the block's largest value within 448.  Scaling by
a power of two rounds nothing, so a value is off by at most half a step of
e4m3: 2^-4 relative, or 2^-10 of the scale where it is that small.  8-bit rows
take half the memory and bandwidth of bfloat16.

Every function runs on the current stream of the tensors' device, allocates
from torch's allocator, and does not synchronise.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Union

import torch

from .softmax import _aligned, _ceil, _native, _place, _rows

BLOCK = 128


class Fp8Rows(NamedTuple):
    """``values`` float8_e4m3fn [R, K] and ``scales`` float8_e8m0fnu
    [R, ceil(K / 128)]: element (r, k) stands for
    values[r, k] * scales[r, k // 128].  Scales are from 2^-126 to 2^127;
    beyond that they are taken as the nearest of those."""
    values: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def nbytes(self) -> int:
        return (self.values.untyped_storage().nbytes()
                + self.scales.untyped_storage().nbytes())


def _check_float(name: str, x) -> None:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(x).__name__}")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{name} must be [rows, columns] with at least one "
                         f"column, got {list(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported dtype {x.dtype}: float32 or bfloat16")
    if x.shape[0] > 2 ** 31 - 1024 or x.shape[1] > 1 << 24:
        raise ValueError("at most 2^31 - 1024 rows of 2^24 columns")
    if not x.is_cuda:
        raise RuntimeError(f"the 8-bit kernels run on the GPU: move {name} "
                           "there")


def _check_rows(name: str, q) -> Fp8Rows:
    if not isinstance(q, Fp8Rows):
        raise TypeError(f"{name} must be Fp8Rows, got {type(q).__name__}")
    values, scales = q
    if values.dtype != torch.float8_e4m3fn or \
            scales.dtype != torch.float8_e8m0fnu:
        raise TypeError(f"{name} must hold float8_e4m3fn values and "
                        f"float8_e8m0fnu scales, got {values.dtype} and "
                        f"{scales.dtype}")
    if values.dim() != 2 or values.shape[1] < 1 or \
            list(scales.shape) != [values.shape[0],
                                   _ceil(values.shape[1], BLOCK)]:
        raise ValueError(f"{name}: {list(values.shape)} values need one scale "
                         f"for every {BLOCK} columns, got "
                         f"{list(scales.shape)}")
    if values.shape[0] > 2 ** 31 - 1024 or values.shape[1] > 1 << 24:
        raise ValueError("at most 2^31 - 1024 rows of 2^24 columns")
    if not (values.is_cuda and scales.is_cuda):
        raise RuntimeError(f"the 8-bit kernels run on the GPU: move {name} "
                           "there")
    if values.device != scales.device:
        raise RuntimeError(f"{name}: values on {values.device}, scales on "
                           f"{scales.device}")
    return Fp8Rows(_rows(values), _rows(scales))


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """Rows [R, K] of float32 or bfloat16 in 8 bits.  Rows of the result start
    at multiples of 16 bytes.  A block's scale is the smallest power of two in
    2^-120 .. 2^120 that keeps its finite values within 448 (within 240 at
    2^120, where 256 would be past float32); what is not finite becomes
    NaN."""
    _check_float("x", x)
    x = _rows(x.detach())
    r, k = x.shape
    held = torch.empty((r, _ceil(k, 16) * 16), dtype=torch.uint8,
                       device=x.device)
    scales = torch.empty((r, _ceil(k, BLOCK)), dtype=torch.uint8,
                         device=x.device)
    _native().quantize_rows(
        x.data_ptr(), x.stride(0), r, k, int(x.dtype == torch.bfloat16),
        held.data_ptr(), held.shape[1], scales.data_ptr(),
        scales.shape[1], 0, *_place(x.device))
    return Fp8Rows(held.view(torch.float8_e4m3fn)[:, :k],
                   scales.view(torch.float8_e8m0fnu))


def dequantize_rows(q: Fp8Rows, dtype: torch.dtype = torch.float32
                    ) -> torch.Tensor:
    """The values that 8-bit rows stand for, exactly: bfloat16 holds them as
    float32 does for scales from 2^-124 on (quantize_rows makes none below
    2^-120), and rounds what smaller ones leave below 2^-133."""
    q = _check_rows("q", q)
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported dtype {dtype}: float32 or bfloat16")
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    _native().dequantize_rows(
        q.values.data_ptr(), q.values.stride(0), q.scales.data_ptr(),
        q.scales.stride(0), q.shape[0], q.shape[1],
        int(dtype == torch.bfloat16), out.data_ptr(), out.shape[1],
        *_place(q.device))
    return out


def matmul_rows(a: Union[torch.Tensor, Fp8Rows], b: Fp8Rows,
                col_scale: Optional[torch.Tensor] = None,
                out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[M, K] rows times [N, K] rows, transposed: out[m, n] = <a_m, b_n>, times
    ``col_scale[n]`` (float32 [N]) where it is given, as [M, N] of ``out_dtype``
    (float32 or bfloat16).  ``a`` is held in 8 bits like ``b``; rows of floats
    are brought to that first.  Products of what dequantize_rows gives as
    bfloat16 are exact, and sums are in 32 bits."""
    b = _check_rows("b", b)
    if isinstance(a, Fp8Rows):
        a = _check_rows("a", a)
    else:
        _check_float("a", a)
    m, k = a.shape
    n = b.shape[0]
    if b.shape[1] != k:
        raise ValueError(f"a has {k} columns, b has {b.shape[1]}")
    if k > 1 << 20:
        raise ValueError("at most 2^20 columns")
    if a.device != b.device:
        raise RuntimeError(f"a is on {a.device}, b on {b.device}")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"unsupported out_dtype {out_dtype}: float32 or "
                        "bfloat16")
    if col_scale is not None:
        if not isinstance(col_scale, torch.Tensor):
            raise TypeError("col_scale must be a tensor, got "
                            f"{type(col_scale).__name__}")
        if col_scale.dtype != torch.float32 or \
                list(col_scale.shape) != [n]:
            raise ValueError(f"col_scale must be float32 [{n}], got "
                             f"{col_scale.dtype} {list(col_scale.shape)}")
        if col_scale.device != b.device:
            raise RuntimeError(f"col_scale is on {col_scale.device}, b on "
                               f"{b.device}")
        col_scale = col_scale.detach().contiguous()
    out = torch.empty((m, n), dtype=out_dtype, device=b.device)
    values, scales = b.values, b.scales.contiguous()
    if scales.data_ptr() % 4:
        scales = scales.clone()
    if not _aligned(values):
        values = torch.empty((n, _ceil(k, 16) * 16), dtype=torch.uint8,
                             device=b.device)
        values[:, :k] = b.values.view(torch.uint8)
    # for wide rows: the scales by block of columns, or a piece of the table
    turned = wide = None
    piece = n
    if k > 320 and m > 160:
        piece = max(256, (64 << 20) // (_ceil(k, 64) * 128) // 256 * 256)
        wide = torch.empty(min(piece, n) * _ceil(k, 64) * 64,
                           dtype=torch.bfloat16, device=b.device)
    elif k > 320 and not (m <= 16 and k <= 2048):
        turned = torch.empty(_ceil(k, BLOCK) * _ceil(n, 256) * 256,
                             dtype=torch.uint8, device=b.device)
    ld = _ceil(k, 8) * 8
    held = torch.empty((m, ld), dtype=torch.bfloat16, device=b.device)
    native, place = _native(), _place(b.device)
    if isinstance(a, Fp8Rows):
        native.dequantize_rows(
            a.values.data_ptr(), a.values.stride(0), a.scales.data_ptr(),
            a.scales.stride(0), m, k, 1, held.data_ptr(), ld, *place)
    else:
        a = _rows(a.detach())
        native.quantize_rows(
            a.data_ptr(), a.stride(0), m, k,
            int(a.dtype == torch.bfloat16), held.data_ptr(), ld, 0, 0, 1,
            *place)
    native.matmul_rows(
        held.data_ptr(), ld, m, values.data_ptr(), values.stride(0),
        scales.data_ptr(), scales.stride(0), n, k,
        0 if col_scale is None else col_scale.data_ptr(), out.data_ptr(),
        int(out_dtype == torch.bfloat16),
        0 if turned is None else turned.data_ptr(),
        0 if wide is None else wide.data_ptr(), piece, *place)
    return out
