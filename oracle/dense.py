"""Linears with an epilogue in 64 bits -- ``act(x w^T + bias)``, gated or not,
``+ residual`` -- and how far a float32 computation rounded once may be from
them."""

from __future__ import annotations

import torch

U = 2.0 ** -24      # half a float32 step
TINY = 2.0 ** -120  # exponentials below float32's range come out as 0


def act(z, name):
    """``(act(z), relative error of computing it in float32, largest slope)``."""
    if name is None:
        return z, torch.zeros_like(z), 1.0
    if name == "relu":
        return z.clamp_min(0), torch.zeros_like(z), 1.0
    if name == "silu":
        # exp(-z) from a rounded exponent: an error of |z| steps; four operations behind it
        return z * torch.sigmoid(z), (2 * z.abs() + 8) * U, 1.1
    if name == "gelu":
        # Phi(-|z|) = exp(-z^2 / 2) times a polynomial (9.4e-8 of its value, 8 steps of Horner's rule); the
        # exponent holds four roundings
        return z * torch.special.ndtr(z), (2 * z * z + 16) * U, 1.13
    if name == "gelu_tanh":
        s = 2 * (2 / torch.pi) ** 0.5 * (z + 0.044715 * z ** 3)
        return z * torch.sigmoid(s), (6 * s.abs() + 8) * U, 1.13
    raise ValueError(name)


def linear(x, w, bias=None, name=None, gated=False, residual=None):
    """``(y float64, bound)``; ``bound(y_dtype)`` is the largest distance, element by element, of the result
    computed with float32 sums and rounded once."""
    K = x.shape[1]
    x, w = x.double(), w.double()
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    # at most K / 4 accumulations one after the other on the matrix cores, 32 inside an instruction, the waves'
    # and splits' partial sums (8 + 16) and the bias
    off = (K / 4 + 64) * U * size
    N = z.shape[1] // 2 if gated else z.shape[1]
    y, rel, slope = act(z[:, :N], name)
    err = slope * off[:, :N] + y.abs() * rel + TINY
    if gated:
        up = z[:, N:]
        err = err * (up.abs() + off[:, N:]) + (y.abs() + err) * off[:, N:] + U * (y * up).abs()
        y = y * up
    if residual is not None:
        y = y + residual.double()
        err = err + U * (y.abs() + err)

    def bound(y_dtype):
        f = torch.finfo(y_dtype)
        return err + f.eps / 2 * (y.abs() + err) + f.smallest_normal * f.eps

    return y, bound


def grouped(x, offsets, w, bias=None, name=None, gated=False):
    """:func:`linear` of the rows of each expert; zeros from ``offsets[-1]`` on."""
    N = w.shape[1] // 2 if gated else w.shape[1]
    y = torch.zeros((x.shape[0], N), dtype=torch.float64)
    parts = []
    for e in range(w.shape[0]):
        b, n = int(offsets[e]), int(offsets[e + 1])
        if n > b:
            y[b:n], bound = linear(x[b:n], w[e], bias[e] if bias is not None else None, name, gated)
            parts.append((b, n, bound))

    def bound(y_dtype):
        t = torch.zeros_like(y)
        for b, n, f in parts:
            t[b:n] = f(y_dtype)
        return t

    return y, bound
