"""RMS norm with the residual's addition and 8-bit rows, on the CPU: the codes
in float32 as defined (they are exact functions of ``p = s * w``), the row's
statistics and everything scaled by them in 64 bits."""

from __future__ import annotations

import torch

TINY = 1e-30


def rms_norm(x, w, eps, residual=None):
    """``(s float32, p float32, rstd float64 [..., 1], y float64)``."""
    s = x.float() if residual is None else x.float() + residual.float()
    rstd = 1.0 / (s.double().square().mean(-1, keepdim=True) + eps).sqrt()
    p = s * w.float()
    return s, p, rstd, s.double() * w.double() * rstd


def fp8_rows(p, rstd):
    """``(codes uint8 [..., H], scale float64 [..., H/128])``."""
    b = p.reshape(*p.shape[:-1], -1, 128)
    m = torch.nan_to_num(b.abs(), nan=0.0, posinf=float("inf")).amax(-1, keepdim=True).clamp_min(TINY)
    q = (b * (torch.full_like(m, 448.0) / m)).to(torch.float8_e4m3fn)
    return q.view(torch.uint8).reshape(p.shape), (m.double() * rstd.unsqueeze(-1) / 448).squeeze(-1)


def int8_rows(p, rstd):
    """``(codes int8 [..., H], scale float64 [...])``."""
    m = torch.nan_to_num(p.abs(), nan=0.0, posinf=float("inf")).amax(-1, keepdim=True).clamp_min(TINY)
    q = torch.nan_to_num((p * (torch.full_like(m, 127.0) / m)).round(), nan=0.0).clamp(-127, 127)
    return q.to(torch.int8), (m.double() * rstd / 127).squeeze(-1)
