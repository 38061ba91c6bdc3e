"""Low-rank adapters of many requests in 64 bits: ``y[t] += scale[i] * B_i
(A_i x[t])`` with ``i = index[t]``, and how far a float32 computation may be
from it."""

from __future__ import annotations

import torch


def add(y, x, a, b, index, scale=None, rank=None):
    """``(y float64, bound)``: ``bound(y_dtype, w_dtype)`` is the largest
    distance, element by element, of the result computed with float32
    products and sums, ``p`` held in parts of the adapters' type, and y
    rounded once."""
    L, R, K = a.shape
    out = y.double()
    inner = torch.zeros_like(out)   # sum_r |b| |scale| sum_k |x a|: rounding of the first product's sums
    part = torch.zeros_like(out)    # sum_r |b| |p|: relative rounding of p's parts and the second product
    top = torch.zeros_like(out)     # sum_r |b| max|p|: f16 parts are relative to the row's largest
    for i in index.unique().tolist():
        if not 0 <= i < L:
            continue
        at = (index == i).nonzero().view(-1)
        r = min(max(int(rank[i]), 0), R) if rank is not None else R
        g = float(scale[i]) if scale is not None else 1.0
        ai, bi, xi = a[i, :r].double(), b[i, :, :r].double(), x[at].double()
        p = g * (xi @ ai.t())
        out[at] += p @ bi.t()
        inner[at] = abs(g) * (xi.abs() @ ai.abs().t()) @ bi.abs().t()
        part[at] = p.abs() @ bi.abs().t()
        if r:
            top[at] = p.abs().amax(1, keepdim=True) * bi.abs().sum(1)

    def bound(y_dtype, w_dtype):
        u = 2.0 ** -24
        # a sum of n products on the matrix cores: at most n / 4 accumulations one after the other, up to 32 inside
        # an instruction, and the waves' and splits' partial sums (4 + 64)
        tol = (K / 4 + 100) * u * inner + (3 * R / 4 + 32) * u * part + 2 * u * out.abs()
        if w_dtype == torch.float16:
            tol = tol + 2.0 ** -21 * top            # two parts of 11 bits, the row scaled by its largest
        else:
            # two parts of 8 bits (each leaves half a step, 2^-9 of what it holds), three under a float32 y
            tol = tol + (2.0 ** -26 if y_dtype == torch.float32 else 2.0 ** -17) * part
        if y_dtype != torch.float32:
            tol = tol + torch.finfo(y_dtype).eps / 2 * (out.abs() + tol)
            tol = tol + torch.finfo(y_dtype).smallest_normal * torch.finfo(y_dtype).eps  # subnormal y
        return tol

    return out, bound
