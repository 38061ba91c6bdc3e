"""Tokens sorted by expert and back, and the gradients, in plain loops and 64
bits."""

from __future__ import annotations

import torch


def plan(ids, E):
    """``(position int32 [T, k], offsets int32 [E + 1])``."""
    T, k = ids.shape
    key = [int(i) if 0 <= int(i) < E else E for i in ids.reshape(-1).tolist()]
    order = sorted(range(T * k), key=lambda a: (key[a], a))
    position = torch.empty(T * k, dtype=torch.int32)
    for row, a in enumerate(order):
        position[a] = row if key[a] < E else ~row
    offsets = [sum(v < e for v in key) for e in range(E + 1)] if T * k <= 4096 else None
    if offsets is None:
        counts = torch.bincount(torch.tensor(key), minlength=E + 1)[:E]
        offsets = [0] + torch.cumsum(counts, 0).tolist()
    return position.view(T, k), torch.tensor(offsets, dtype=torch.int32)


def permute(x, position):
    T, k = position.shape
    rows = torch.zeros((T * k, x.shape[1]), dtype=x.dtype)
    for s in range(k):
        kept = position[:, s] >= 0
        rows[position[kept, s].long()] = x[kept]
    return rows


def unpermute(rows, position, weights=None):
    """``(y float64, bound)``: float32 products and sums in slot order, rounded once."""
    T, k = position.shape
    y = torch.zeros((T, rows.shape[1]), dtype=torch.float64)
    size = torch.zeros_like(y)
    for s in range(k):
        kept = position[:, s] >= 0
        part = rows[position[kept, s].long()].double()
        if weights is not None:
            part = part * weights[kept, s].double()[:, None]
        y[kept] += part
        size[kept] += part.abs()

    def bound(dtype):
        f = torch.finfo(dtype)
        err = (k + 1) * 2.0 ** -24 * size  # each sum (and a product's own rounding, where it is not fused)
        return err + f.eps / 2 * (y.abs() + err) + f.smallest_normal * f.eps

    return y, bound


def unpermute_backward(dy, rows, position, weights):
    """``(d_rows float64, d_weights float64, bound of d_weights)``."""
    T, k = position.shape
    d_rows = torch.zeros((T * k, rows.shape[1]), dtype=torch.float64)
    d_weights = torch.zeros((T, k), dtype=torch.float64)
    size = torch.zeros((T, k), dtype=torch.float64)
    for s in range(k):
        kept = position[:, s] >= 0
        at = position[kept, s].long()
        g = dy[kept].double()
        d_rows[at] = weights[kept, s].double()[:, None] * g
        prod = rows[at].double() * g
        d_weights[kept, s] = prod.sum(1)
        size[kept, s] = prod.abs().sum(1)
    # a lane adds at most H / 64 / 4 pieces' values one after the other, then 6 + 4 sums
    return d_rows, d_weights, (rows.shape[1] / 64 + 32) * 2.0 ** -24 * size + 1e-40
