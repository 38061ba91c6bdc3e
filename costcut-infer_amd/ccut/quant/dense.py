"""Linears whose weights a checkpoint keeps in 16 bits (``ccq_dense_linear``,
``ccq_dense_linear_grouped``), with bias, activation and residual in the
product's own kernel:

    z = x @ w.T + bias
    y = act(z) + residual                         w [N, K]
    y = act(z[..., :N]) * z[..., N:] + residual   w [2N, K], gated=True

in float32, ``y`` rounded once.  :func:`linear` is for a batch of rows,
:func:`linear_grouped` for rows sorted by expert (``blocks.moe.moe_permute``).
The weights of a gated product are the gate's rows followed by the up rows,
``torch.cat([w_gate, w_up], -2)``.  Values only: no gradients."""

from __future__ import annotations

import torch

from ccut._dev import DTYPE_CODE, empty_strided, is_current, raw_stream, rows_overlap
from ccut._lib import ACTIVATIONS, DENSE_ARGS, check, lib

__all__ = ["linear", "linear_grouped"]

_HALF = (torch.bfloat16, torch.float16)
_pack = DENSE_ARGS.pack
MAX_ROWS, MAX_SIDE, MAX_EXPERTS = 1 << 20, 1 << 20, 1024
# batches of up to this many rows take no scratch
_BARE_ROWS = 16


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """A [rows, width] view of ``t`` (or a dense copy) and its row stride."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[0] <= 1:
        return (t if t.stride(1) == 1 else t.contiguous()), t.shape[1]
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, t.stride(0)


def _dense(x, offsets, w, bias, act, gated: bool, residual, out, out_dtype):
    index = x.get_device()
    if not is_current(index):
        with torch.cuda.device(index):
            return _dense(x, offsets, w, bias, act, gated, residual, out, out_dtype)
    dtype, shape = x.dtype, x.shape
    if dtype not in _HALF:
        raise ValueError(f"rows must be float16 or bfloat16, got {dtype}")
    if w.dtype != dtype or w.get_device() != index:
        raise ValueError(f"w is {w.dtype} on {w.device}, x {dtype} on {x.device}")
    dims = 2 if offsets is None else 3
    if w.dim() != dims or not shape or (offsets is not None and len(shape) != 2):
        raise ValueError(f"x {tuple(shape)} and w {tuple(w.shape)}: must be "
                         f"{'[..., K] and [N, K]' if offsets is None else '[rows, K] and [experts, N, K]'}")
    K, W = shape[-1], w.shape[-2]
    N = W >> 1 if gated else W
    if w.shape[-1] != K or not 1 <= K <= MAX_SIDE or not 1 <= N <= MAX_SIDE or (gated and W & 1):
        raise ValueError(f"x {tuple(shape)} and w {tuple(w.shape)}: K must agree, 1 <= K, N <= {MAX_SIDE}"
                         f"{', w of a gated product has 2 N rows' if gated else ''}")
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"act={act!r}: one of {', '.join(map(repr, ACTIVATIONS))}")
    E = 0
    if offsets is not None:
        E = w.shape[0]
        if not 1 <= E <= MAX_EXPERTS:
            raise ValueError(f"w {tuple(w.shape)}: 1 to {MAX_EXPERTS} experts")
        if offsets.dtype != torch.int32 or tuple(offsets.shape) != (E + 1,) or offsets.get_device() != index:
            raise ValueError(f"offsets must be int32 [{E + 1}] on {x.device}, got {offsets.dtype} "
                             f"{tuple(offsets.shape)} on {offsets.device}")
        if not offsets.is_contiguous():
            offsets = offsets.contiguous()
    if not w.is_contiguous():
        w = w.contiguous()
    bp = bcode = 0
    if bias is not None:
        bcode = DTYPE_CODE.get(bias.dtype)
        if bcode is None or bias.shape != w.shape[:-1] or bias.get_device() != index:
            raise ValueError(f"bias must be float32, float16 or bfloat16 {tuple(w.shape[:-1])} on {x.device}, got "
                             f"{bias.dtype} {tuple(bias.shape)} on {bias.device}")
        if not bias.is_contiguous():
            bias = bias.contiguous()
        bp = bias.data_ptr()
    x2, ldx = (x, K) if len(shape) == 2 and x.is_contiguous() else _rows(x)
    M = x2.shape[0]
    if M > MAX_ROWS:
        raise ValueError(f"{M} rows: at most {MAX_ROWS}")
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else dtype
    ycode = DTYPE_CODE.get(out_dtype)
    if ycode is None:
        raise ValueError(f"y must be float32, float16 or bfloat16, got {out_dtype}")
    y_shape = shape[:-1] + (N,)
    xp = x2.data_ptr()
    if out is None:
        y = empty_strided((M, N), (N, 1), out_dtype)
        yp, ldy = y.data_ptr(), N
        out = y if len(shape) == 2 else y.view(y_shape)
    else:
        if out.dtype != out_dtype or out.shape != y_shape or out.get_device() != index:
            raise ValueError(f"out must be {out_dtype} {tuple(y_shape)} on {x.device}, got {out.dtype} "
                             f"{tuple(out.shape)} on {out.device}")
        y2, ldy = _rows(out)
        yp = y2.data_ptr()
        if yp != out.data_ptr():  # a copy, so not a view that could be written
            raise ValueError("out must hold its rows one after the other, each of them dense")
        if rows_overlap(yp, ycode, ldy, N, xp, DTYPE_CODE[dtype], ldx, K, M):
            raise ValueError("out overlaps x")
        end = yp + ((M - 1) * ldy + N) * out.element_size()
        for t in (w, bias, offsets):
            if t is not None and M and t.data_ptr() < end and yp < t.data_ptr() + t.numel() * t.element_size():
                raise ValueError("out overlaps w, bias or offsets")
    rp = ldr = 0
    if residual is not None:
        if residual.dtype != out_dtype or residual.shape != y_shape or residual.get_device() != index:
            raise ValueError(f"residual must be {out_dtype} {tuple(y_shape)} on {x.device}, got {residual.dtype} "
                             f"{tuple(residual.shape)} on {residual.device}")
        r2, ldr = _rows(residual)
        rp = r2.data_ptr()
        if (rp, ldr) != (yp, ldy) and rows_overlap(yp, ycode, ldy, N, rp, ycode, ldr, N, M):
            raise ValueError("out overlaps residual and is not residual")
    if M == 0:
        return out
    handle = lib()
    wp, op = w.data_ptr(), 0
    run, size = handle.ccq_dense_linear, handle.ccq_dense_linear_workspace_size
    scratch = M > _BARE_ROWS
    if offsets is not None:
        op, run, size = offsets.data_ptr(), handle.ccq_dense_linear_grouped, handle.ccq_dense_linear_grouped_workspace_size
        scratch = (K | ldx) & 7 or (xp | wp) & 15  # (aligned groups take none)
    sp = nbytes = 0
    tail = (ldx, ldr, ldy, M, K, N, E, DTYPE_CODE[dtype], bcode, ycode, code, gated)
    if scratch:
        nbytes = size(_pack(xp, wp, bp, rp, yp, op, 0, 0, 0, *tail))
        if nbytes:  # this call's own, so that calls on several streams or in several graphs do not share it
            scratch = empty_strided((nbytes,), (1,), torch.uint8)
            sp = scratch.data_ptr()
    rc = run(_pack(xp, wp, bp, rp, yp, op, sp, raw_stream(index), nbytes, *tail))
    if rc:
        check(rc, "ccq_dense_linear" if offsets is None else "ccq_dense_linear_grouped")
    return out


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *, act: str | None = None,
           gated: bool = False, residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``act(x @ w.T + bias) + residual`` for device rows ``x [..., K]`` and
    ``w [N, K]``, both float16 or both bfloat16 (gated: ``w [2N, K]``,
    ``act`` of the first N columns times the others).  ``act``: None,
    ``"relu"``, ``"gelu"``, ``"gelu_tanh"`` or ``"silu"``; ``bias`` of any
    float type; ``residual`` of the output's type (``out_dtype``, default
    ``out``'s or x's) and shape.  ``out`` is written where given: it may be
    ``residual``, but no other view of it or of ``x``, and must not lie
    around ``w`` or ``bias``.  Rows may have any stride; ``w`` and ``bias``
    that are not dense are copied."""
    return _dense(x, None, w, bias, act, bool(gated), residual, out, out_dtype)


def linear_grouped(x: torch.Tensor, offsets: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None, *,
                   act: str | None = None, gated: bool = False, out: torch.Tensor | None = None,
                   out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """:func:`linear` of rows sorted by expert: rows ``offsets[e]`` to
    ``offsets[e + 1]`` of ``x [rows, K]`` with ``w[e]`` of ``w [E, N, K]``
    (gated: ``[E, 2N, K]``) and ``bias[e]``.  ``offsets [E + 1]`` (int32, on
    the device, rising from 0, as ``moe_permute`` returns them; the host does
    not read it).  Rows of the result from ``offsets[E]`` on are zeros; others
    that no two of the offsets hold between them are not written."""
    if offsets is None:
        raise ValueError("linear_grouped needs offsets")
    return _dense(x, offsets, w, bias, act, bool(gated), None, out, out_dtype)
