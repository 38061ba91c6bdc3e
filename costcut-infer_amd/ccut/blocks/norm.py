"""RMS norm with the residual's addition on the GPU, and its output in the
8-bit formats that the quantized linears multiply (``ccq_rms_norm``).

Per row, in float32: ``s = x + residual``, ``y = s * rsqrt(mean(s^2) + eps) *
weight``.  One pass over the rows writes the sum (the next residual), the
8-bit rows with their scales, and, where asked, the normalized rows
themselves (for a router or adapters beside a quantized projection).

- :func:`rms_norm`: the normalized rows (the reference's ``rms_norm``,
  ``python/ccut/blocks/norm.py:14``, with the addition before it);
- :func:`rms_norm_fp8`: e4m3 codes, a scale per row and 128 columns, for
  ``quant.fp8_block.linear_quantized``;
- :func:`rms_norm_int8`: int8 codes, a scale per row, for
  ``quant.int8.int8_linear``.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ccut import _dev
from ccut._dev import DTYPE_CODE, empty_strided, is_current, raw_stream, rows_overlap
from ccut._lib import CCQ_Q_FP8_BLOCK, CCQ_Q_INT8_ROW, CCQ_Q_NONE, RMS_NORM_ARGS, check, lib

_U8, _I8, _F32 = torch.uint8, torch.int8, torch.float32
_pack = RMS_NORM_ARGS.pack

__all__ = ["rms_norm", "rms_norm_fp8", "rms_norm_int8", "QuantizedRows"]

MAX_H = 32768
MAX_EPS = 3.4e38  # a float32


class QuantizedRows(NamedTuple):
    """8-bit rows: ``q`` (uint8 e4m3 codes, or int8) of x's shape, ``scale``
    float32 (``[..., H/128]`` for FP8, ``[...]`` for INT8); ``y`` the
    normalized rows in x's type (with ``normed=True``), ``residual`` the sum
    ``x + residual`` in x's type (where a residual was given)."""

    q: torch.Tensor
    scale: torch.Tensor
    y: torch.Tensor | None
    residual: torch.Tensor | None


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """A [rows, H] view of ``t`` and its row stride (a single row's stride has
    no meaning and may be any)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[0] <= 1:
        return (t if t.stride(1) == 1 else t.contiguous()), t.shape[1]
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, t.stride(0)


def _unlike(t: torch.Tensor, what: str, x: torch.Tensor) -> ValueError:
    return ValueError(f"{what} is {t.dtype} {tuple(t.shape)} on {t.device}; x is {x.dtype} {tuple(x.shape)} on "
                      f"{x.device}")


def _norm(x: torch.Tensor, weight, eps: float, residual, residual_out, normed: bool, y_dtype, q_fmt: int):
    # (a decode call is 3 us on the GPU: what is asked of torch here is what counts)
    index = x.get_device()
    if not is_current(index):
        with torch.cuda.device(index):
            return _norm(x, weight, eps, residual, residual_out, normed, y_dtype, q_fmt)
    dtype, shape = x.dtype, x.shape
    code = DTYPE_CODE.get(dtype)
    if code is None:
        raise ValueError(f"rows must be float32, float16 or bfloat16, got {dtype}")
    H = shape[-1] if shape else 0
    if not 1 <= H <= MAX_H:
        raise ValueError(f"rows must be [..., H] with 1 <= H <= {MAX_H}, got {tuple(shape)}")
    if q_fmt == CCQ_Q_FP8_BLOCK and H & 127:
        raise ValueError(f"FP8 rows need H % 128 == 0, got H={H}")
    if not 0 < eps < MAX_EPS:
        raise ValueError(f"eps must be positive and finite, got {eps}")
    wcode = DTYPE_CODE.get(weight.dtype)
    if wcode is None or weight.dim() != 1 or weight.numel() != H or weight.get_device() != index:
        raise ValueError(f"weight must be [{H}] float32, float16 or bfloat16 on {x.device}, got {weight.dtype} "
                         f"{tuple(weight.shape)} on {weight.device}")
    if not weight.is_contiguous():
        weight = weight.contiguous()
    flat = len(shape) == 2
    x2, ldx = (x, H) if flat and x.is_contiguous() else _rows(x)
    T = shape[0] if flat else x2.shape[0]
    size, strides = (T, H), (H, 1)
    q = scale = y = None
    rp = op = yp = qp = sp = ldr = ldo = ycode = 0
    if residual is not None:
        if residual.dtype != dtype or residual.shape != shape or residual.get_device() != index:
            raise _unlike(residual, "residual", x)
        r2, ldr = (residual, H) if flat and residual.is_contiguous() else _rows(residual)
        rp = r2.data_ptr()
        if residual_out is None:
            residual_out = empty_strided(size, strides, dtype)
            op, ldo = residual_out.data_ptr(), H
            if not flat:
                residual_out = residual_out.view(shape)
        else:
            if residual_out.dtype != dtype or residual_out.shape != shape or residual_out.get_device() != index:
                raise _unlike(residual_out, "residual_out", x)
            o2, ldo = _rows(residual_out)
            op = o2.data_ptr()
            if op != residual_out.data_ptr():  # a copy, so not a view that could be written
                raise ValueError("residual_out must hold its rows one after the other, each of them dense")
            for p, ld in ((x2.data_ptr(), ldx), (rp, ldr)):
                if (p, ld) != (op, ldo) and rows_overlap(op, code, ldo, H, p, code, ld, H, T):
                    raise ValueError("residual_out overlaps x or residual and is neither")
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    if normed:
        ycode = code if y_dtype is None else DTYPE_CODE[y_dtype]
        y = empty_strided(size, strides, y_dtype or dtype)
        yp = y.data_ptr()
    if q_fmt == CCQ_Q_FP8_BLOCK:
        q = empty_strided(size, strides, _U8)
        scale = empty_strided((T, H >> 7), (H >> 7, 1), _F32)
        qp, sp = q.data_ptr(), scale.data_ptr()
    elif q_fmt == CCQ_Q_INT8_ROW:
        q = empty_strided(size, strides, _I8)
        scale = empty_strided((T,), (1,), _F32)
        qp, sp = q.data_ptr(), scale.data_ptr()
    rc = lib().ccq_rms_norm_packed(_pack(x2.data_ptr(), rp, weight.data_ptr(), op, yp, qp, sp, raw_stream(index), ldx,
                                         ldr, ldo, T, H, code, wcode, ycode, q_fmt, eps))
    if rc:
        check(rc, "ccq_rms_norm")
    if not flat:
        y = y.view(shape) if y is not None else None
        if q is not None:
            q = q.view(shape)
            scale = scale.view(*shape[:-1], H >> 7) if q_fmt == CCQ_Q_FP8_BLOCK else scale.view(shape[:-1])
    return QuantizedRows(q, scale, y, residual_out)


def rms_norm(x, weight, eps: float = 1e-6, *, residual=None, residual_out: torch.Tensor | None = None,
             out_dtype: torch.dtype | None = None):
    """``y = s * rsqrt(mean(s^2) + eps) * weight`` with ``s = x + residual``
    over the last dimension, computed in float32; returns ``y`` (``out_dtype``,
    default x's), or ``(y, s)`` where a residual is given (``s`` in x's type,
    written to ``residual_out``, which may be ``residual`` or ``x`` but no
    other view of their memory).  Host
    arrays are uploaded as float32 and numpy float32 is returned, no other
    ``out_dtype``."""
    if _dev.is_host(x):
        if out_dtype not in (None, torch.float32):
            raise ValueError(f"host rows are returned as float32, not {out_dtype}")

        def up(a):
            return a if a is None else _dev.to_device(a, torch.float32)

        if residual_out is not None:
            raise ValueError("residual_out is for device rows")
        _, _, y, s = _norm(up(x), up(weight), eps, up(residual), None, True, None, CCQ_Q_NONE)
        return _dev.to_host(y) if s is None else (_dev.to_host(y), _dev.to_host(s))
    if out_dtype is not None and out_dtype not in DTYPE_CODE:
        raise ValueError(f"rows must be float32, float16 or bfloat16, got {out_dtype}")
    _, _, y, s = _norm(x, weight, eps, residual, residual_out, True, out_dtype, CCQ_Q_NONE)
    return y if s is None else (y, s)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, residual: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None, normed: bool = False) -> QuantizedRows:
    """:func:`rms_norm` of device rows (H % 128 == 0) to e4m3 codes with a
    scale per row and 128 columns; ``normed`` returns the normalized rows
    (x's type) beside them, from the same pass."""
    return _norm(x, weight, eps, residual, residual_out, normed, None, CCQ_Q_FP8_BLOCK)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, residual: torch.Tensor | None = None,
                  residual_out: torch.Tensor | None = None, normed: bool = False) -> QuantizedRows:
    """:func:`rms_norm` of device rows to int8 codes with a scale per row
    (``amax / 127``; ``quant.int8.quantize_per_token`` keeps the reference's
    factor, which saturates almost every value); ``normed`` as in
    :func:`rms_norm_fp8`."""
    return _norm(x, weight, eps, residual, residual_out, normed, None, CCQ_Q_INT8_ROW)
