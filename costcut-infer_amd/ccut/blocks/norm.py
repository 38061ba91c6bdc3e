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
from ccut._lib import CCQ_Q_FP8_BLOCK, CCQ_Q_INT8_ROW, CCQ_Q_NONE, call

__all__ = ["rms_norm", "rms_norm_fp8", "rms_norm_int8", "QuantizedRows"]

MAX_H = 32768


class QuantizedRows(NamedTuple):
    """8-bit rows: ``q`` (uint8 e4m3 codes, or int8) of x's shape, ``scale``
    float32 (``[..., H/128]`` for FP8, ``[...]`` for INT8); ``y`` the
    normalized rows in x's type (with ``normed=True``), ``residual`` the sum
    ``x + residual`` in x's type (where a residual was given)."""

    q: torch.Tensor
    scale: torch.Tensor
    y: torch.Tensor | None
    residual: torch.Tensor | None


def _rows(t: torch.Tensor, what: str, like: torch.Tensor) -> torch.Tensor:
    """A [rows, H] view of ``t`` for the kernel, which takes row strides."""
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{what} is {t.dtype} {tuple(t.shape)} on {t.device}; x is {like.dtype} "
                         f"{tuple(like.shape)} on {like.device}")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] <= 1) else t.contiguous()


def _ld(t: torch.Tensor) -> int:
    """The row stride (a single row's stride has no meaning and may be any)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _norm(x: torch.Tensor, weight, eps: float, residual, residual_out, y_dtype, q_fmt: int):
    if not x.is_cuda:
        raise ValueError(f"Expected a cuda device, but got: {x.device}")
    if x.get_device() != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return _norm(x, weight, eps, residual, residual_out, y_dtype, q_fmt)
    if x.dtype not in _dev.DTYPE_CODE:
        raise ValueError(f"rows must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_H:
        raise ValueError(f"rows must be [..., H] with 1 <= H <= {MAX_H}, got {tuple(x.shape)}")
    H = x.shape[-1]
    if q_fmt == CCQ_Q_FP8_BLOCK and H % 128:
        raise ValueError(f"FP8 rows need H % 128 == 0, got H={H}")
    if not eps > 0 or eps == float("inf"):
        raise ValueError(f"eps must be positive and finite, got {eps}")
    if weight.shape != (H,) or weight.dtype not in _dev.DTYPE_CODE or weight.device != x.device:
        raise ValueError(f"weight must be [{H}] float32, float16 or bfloat16 on {x.device}, got {weight.dtype} "
                         f"{tuple(weight.shape)} on {weight.device}")
    weight = weight.contiguous()
    x2 = _rows(x, "x", x)
    T = x2.shape[0]
    r2 = o2 = None
    if residual is not None:
        r2 = _rows(residual, "residual", x)
        if residual_out is None:
            residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        o2 = _rows(residual_out, "residual_out", x)
        if o2.data_ptr() != residual_out.data_ptr():  # a copy, so not a view that could be written
            raise ValueError("residual_out must hold its rows one after the other, each of them dense")
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    y = torch.empty(x.shape, dtype=y_dtype, device=x.device) if y_dtype is not None else None
    q = scale = None
    if q_fmt == CCQ_Q_FP8_BLOCK:
        q = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
        scale = torch.empty((*x.shape[:-1], H // 128), dtype=torch.float32, device=x.device)
    elif q_fmt == CCQ_Q_INT8_ROW:
        q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    call("ccq_rms_norm", x2.data_ptr(), _dev.DTYPE_CODE[x.dtype], _ld(x2),
         r2.data_ptr() if r2 is not None else None, _ld(r2) if r2 is not None else 0,
         weight.data_ptr(), _dev.DTYPE_CODE[weight.dtype], eps,
         o2.data_ptr() if o2 is not None else None, _ld(o2) if o2 is not None else 0,
         y.data_ptr() if y is not None else None, _dev.DTYPE_CODE[y_dtype] if y is not None else 0, q_fmt,
         q.data_ptr() if q is not None else None, scale.data_ptr() if scale is not None else None, T, H,
         _dev.stream_ptr(x.device))
    return q, scale, y, residual_out


def rms_norm(x, weight, eps: float = 1e-6, *, residual=None, residual_out: torch.Tensor | None = None,
             out_dtype: torch.dtype | None = None):
    """``y = s * rsqrt(mean(s^2) + eps) * weight`` with ``s = x + residual``
    over the last dimension, computed in float32; returns ``y`` (``out_dtype``,
    default x's), or ``(y, s)`` where a residual is given (``s`` in x's type,
    written to ``residual_out``, which may be ``residual`` or ``x``).  Host
    arrays are uploaded as float32 and numpy float32 is returned."""
    if _dev.is_host(x):
        def up(a):
            return a if a is None else _dev.to_device(a, torch.float32)

        if residual_out is not None:
            raise ValueError("residual_out is for device rows")
        _, _, y, s = _norm(up(x), up(weight), eps, up(residual), None, torch.float32, CCQ_Q_NONE)
        return _dev.to_host(y) if s is None else (_dev.to_host(y), _dev.to_host(s))
    y_dtype = out_dtype or x.dtype
    if y_dtype not in _dev.DTYPE_CODE:
        raise ValueError(f"rows must be float32, float16 or bfloat16, got {y_dtype}")
    _, _, y, s = _norm(x, weight, eps, residual, residual_out, y_dtype, CCQ_Q_NONE)
    return y if s is None else (y, s)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, residual: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None, normed: bool = False) -> QuantizedRows:
    """:func:`rms_norm` of device rows (H % 128 == 0) to e4m3 codes with a
    scale per row and 128 columns; ``normed`` returns the normalized rows
    (x's type) beside them, from the same pass."""
    return QuantizedRows(*_norm(x, weight, eps, residual, residual_out, x.dtype if normed else None,
                                CCQ_Q_FP8_BLOCK))


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, *, residual: torch.Tensor | None = None,
                  residual_out: torch.Tensor | None = None, normed: bool = False) -> QuantizedRows:
    """:func:`rms_norm` of device rows to int8 codes with a scale per row
    (``amax / 127``; ``quant.int8.quantize_per_token`` keeps the reference's
    factor, which saturates almost every value); ``normed`` as in
    :func:`rms_norm_fp8`."""
    return QuantizedRows(*_norm(x, weight, eps, residual, residual_out, x.dtype if normed else None,
                                CCQ_Q_INT8_ROW))
