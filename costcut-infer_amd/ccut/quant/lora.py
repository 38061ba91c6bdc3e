"""Low-rank adapters of many requests at once beside one shared projection
(``ccq_lora_add``): ``y[t] += scale[i] * B_i (A_i x[t])`` with ``i =
index[t]``, in place on the projection's output -- ``awq.gemm``,
``fp8_block.linear``, ``int8.int8_linear`` or ``LinearProj.apply`` (which
takes the adapters itself).  Rows without an adapter are left as they are.
Products and sums are float32 and y is rounded once.  The reference serves
one request at a time and has no counterpart."""

from __future__ import annotations

import torch

from ccut import _dev
from ccut._dev import DTYPE_CODE, empty_strided, is_current, raw_stream
from ccut._dev import rows_overlap as _overlap
from ccut._lib import ccq_lora_adapters, check, lib

__all__ = ["LoraAdapters", "add_"]

MAX_ADAPTERS, MAX_RANK, MAX_TOKENS = 1024, 256, 65536


class LoraAdapters:
    """The adapters of one projection, stacked on the device: ``a [L, R, in]``
    and ``b [L, out, R]`` (float16 or bfloat16), ``scale [L]`` (float32; None:
    1 each), ``rank [L]`` (int32; None: R each) -- the ranks of an adapter
    from ``rank[i]`` on are padding, and what they hold is not used.  Dense
    tensors are referred to as they are, so an adapter can be replaced by
    writing into them (on the stream that uses them); others are copied once.
    The tensors themselves stay those of the construction."""

    _FIXED = frozenset(("a", "b", "scale", "rank", "num_adapters", "rank_max", "in_features", "out_features", "device",
                        "_index", "_desc", "_held"))

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale=None, rank=None):
        if not a.is_cuda:
            raise ValueError(f"Expected a cuda device, but got: {a.device}")
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"adapters must be a [L, R, in] and b [L, out, R], got {tuple(a.shape)} and "
                             f"{tuple(b.shape)}")
        if a.dtype != b.dtype or a.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"adapters must both be float16 or bfloat16, got {a.dtype} and {b.dtype}")
        L, R, K = a.shape
        if not (1 <= L <= MAX_ADAPTERS and 1 <= R <= MAX_RANK and K >= 1 and b.shape[1] >= 1):
            raise ValueError(f"adapters a {tuple(a.shape)}, b {tuple(b.shape)}: need 1 to {MAX_ADAPTERS} adapters of "
                             f"rank 1 to {MAX_RANK}, in and out at least 1")
        scale = self._vector(scale, torch.float32, L, a.device, "scale")
        rank = self._vector(rank, torch.int32, L, a.device, "rank")
        if b.device != a.device:
            raise ValueError(f"a on {a.device}, b on {b.device}")
        a, b = a.contiguous(), b.contiguous()
        desc = ccq_lora_adapters(a.data_ptr(), b.data_ptr(), scale.data_ptr() if scale is not None else None,
                                 rank.data_ptr() if rank is not None else None, DTYPE_CODE[a.dtype], L, R, K, b.shape[1])
        self.__dict__.update(a=a, b=b, scale=scale, rank=rank, num_adapters=L, rank_max=R, in_features=K,
                             out_features=b.shape[1], device=a.device, _index=a.get_device(), _desc=desc, _bytes={},
                             _held=[t.untyped_storage() for t in (a, b, scale, rank) if t is not None])

    def __setattr__(self, name: str, value) -> None:
        # the descriptor holds the tensors' addresses: another tensor in their place would not be the one that is read
        if name in self._FIXED:
            raise AttributeError(f"{name}: adapters are replaced by writing into their tensors")
        super().__setattr__(name, value)

    @staticmethod
    def _vector(v, dtype: torch.dtype, L: int, device, what: str) -> torch.Tensor | None:
        if v is None:
            return None
        t = v if isinstance(v, torch.Tensor) else torch.as_tensor(v)
        if tuple(t.shape) != (L,):
            raise ValueError(f"{what} must have one entry per adapter ({L}), got {tuple(t.shape)}")
        return t.to(device=device, dtype=dtype).contiguous()

    def workspace_size(self, xp: int, x_code: int, ldx: int, T: int) -> int:
        """Bytes of scratch that ``add_`` takes for T rows of x at ``xp``."""
        key = (T, x_code, ldx, xp & 15)
        n = self._bytes.get(key)
        if n is None:
            if len(self._bytes) >= 4096:
                self._bytes.clear()
            n = self._bytes[key] = int(lib().ccq_lora_workspace_size(xp, x_code, ldx, T, self._desc))
        return n


def _rows(t: torch.Tensor, width: int, what: str) -> torch.Tensor:
    if t.dtype not in DTYPE_CODE:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    if t.dim() < 1 or t.shape[-1] != width:
        raise ValueError(f"{what} must be [..., {width}], got {tuple(t.shape)}")
    return t if t.dim() == 2 else t.reshape(-1, width)


def _dense_rows(t: torch.Tensor) -> bool:
    return t.is_contiguous() or t.stride(1) == 1 and t.stride(0) >= t.shape[1]


def add_(y: torch.Tensor, x: torch.Tensor, adapters: LoraAdapters, index: torch.Tensor) -> torch.Tensor:
    """``y[t] += scale[i] * (x[t] @ a[i].T) @ b[i].T`` with ``i = index[t]``,
    in place; returns ``y``.  ``y [..., out]`` and ``x [..., in]`` (float32,
    float16 or bfloat16 each, rows dense but with any row stride) and ``index
    [...]`` (int64; other whole numbers are converted) are device tensors with
    the same leading dimensions, at most 65536 rows.  An index outside [0, L)
    means no adapter: that row is left as it is.  ``y`` must not overlap
    ``x``.  Repeated calls give the same bits (sums have a fixed
    order)."""
    dev = y.get_device()
    if not is_current(dev):
        with torch.cuda.device(dev):
            return add_(y, x, adapters, index)
    if x.get_device() != dev or index.get_device() != dev or adapters._index != dev:
        raise ValueError(f"y on {y.device}, x on {x.device}, index on {index.device}, adapters on {adapters.device}")
    if x.shape[:-1] != index.shape or y.shape[:-1] != index.shape:
        raise ValueError(f"leading dimensions of y {tuple(y.shape)}, x {tuple(x.shape)} and index "
                         f"{tuple(index.shape)} differ")
    y2, x2 = _rows(y, adapters.out_features, "y"), _rows(x, adapters.in_features, "x")
    yp = y2.data_ptr()
    if y2 is not y and yp != y.data_ptr() or not _dense_rows(y2):
        raise ValueError("y must hold its rows one after the other, each of them dense (it is written in place)")
    if not _dense_rows(x2):
        x2 = x2.contiguous()
    if index.dtype != torch.int64 or not index.is_contiguous():
        if index.dtype not in (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8):
            raise ValueError(f"index must hold whole numbers, got {index.dtype}")
        index = index.to(torch.int64).contiguous()
    T = y2.shape[0]
    if T > MAX_TOKENS:
        raise ValueError(f"{T} rows: at most {MAX_TOKENS}")
    if T == 0:
        return y
    ldx, ldy = (x2.stride(0), y2.stride(0)) if T > 1 else (adapters.in_features, adapters.out_features)
    xp, xcode, ycode = x2.data_ptr(), DTYPE_CODE[x2.dtype], DTYPE_CODE[y2.dtype]
    if _overlap(yp, ycode, ldy, adapters.out_features, xp, xcode, ldx, adapters.in_features, T):
        raise ValueError("y overlaps x")
    nbytes = adapters.workspace_size(xp, xcode, ldx, T)
    wp = None
    if nbytes:  # this call's own scratch, so that calls on several streams or in several graphs do not share it
        ws = empty_strided((nbytes,), (1,), torch.uint8)
        wp = ws.data_ptr()
    rc = lib().ccq_lora_add(xp, xcode, ldx, index.data_ptr(), yp, ycode, ldy, T, adapters._desc, wp, nbytes,
                            raw_stream(dev))
    if rc:
        check(rc, "ccq_lora_add")
    return y
