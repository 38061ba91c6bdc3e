"""Device plumbing shared by the Python front end: tensors in HBM, streams,
dtype codes.  torch is used only for device memory and streams here; every
computation runs in libccq_hip.so."""

from __future__ import annotations

import warnings

import numpy as np
import torch

from ccut._lib import CCQ_BF16, CCQ_F16, CCQ_F32

DTYPE_CODE = {torch.float32: CCQ_F32, torch.float16: CCQ_F16, torch.bfloat16: CCQ_BF16}


# (looking a device up here takes 0.08 us, making its ``type`` string 0.23)
_GPUS = frozenset(torch.device("cuda", i) for i in range(16))


def require_gpu() -> torch.device:
    if not torch.cuda.is_available():
        raise RuntimeError("the quantized expert path runs on a ROCm GPU only (no CPU fallback); "
                           "torch.cuda.is_available() is False")
    return torch.device("cuda", torch.cuda.current_device())


def stream_ptr(device: torch.device | None = None) -> int:
    """The hipStream_t of the device's current torch stream.  Callers hold a
    tensor on the device, so torch is initialised; the raw query is 0.1 us,
    ``torch.cuda.current_stream().cuda_stream`` 2.0-2.8 us of a decode call
    that takes 5 us on the GPU.  A device that is no GPU is refused, as
    ``current_stream`` does: for the calls that take ``x`` as it comes this is
    what keeps a host pointer from a kernel."""
    if device is not None and device not in _GPUS and device.type != "cuda":
        raise ValueError(f"Expected a cuda device, but got: {device}")
    index = device.index if device is not None and device.index is not None else torch.cuda.current_device()
    return raw_stream(index)


def _empty_strided(size, strides, dtype: torch.dtype) -> torch.Tensor:
    return torch.empty_strided(size, strides, dtype=dtype, device="cuda")


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


def _current_device() -> int:
    return torch.cuda.current_device()


# Short cuts inside torch, where this torch has them (one built for the CPU
# lacks some, and they carry no promise), else the public calls above.
# empty_strided: a tensor of uninitialised memory on the current device, by
# (shape, strides, dtype): 0.8 us, torch.empty 1.3-1.6 (a decode call with three
# outputs takes 3-5 us on the GPU).
_guards = getattr(getattr(torch._C, "_dynamo", None), "guards", None)
empty_strided = getattr(_guards, "_empty_strided_cuda", _empty_strided)
raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)  # of a device's index: what stream_ptr asks
current_device = getattr(torch._C, "_cuda_getDevice", _current_device)


def is_current(index: int) -> bool:
    """Whether ``index`` (``Tensor.get_device()``) is the current device; a
    host tensor's -1 is refused.  Callers hold a tensor, so torch is
    initialised: 0.15 us, ``torch.cuda.current_device()`` 0.25."""
    if index < 0:
        raise ValueError("Expected a cuda device, but got: cpu")
    return index == current_device()


def rows_overlap(yp: int, ycode: int, ldy: int, N: int, xp: int, xcode: int, ldx: int, K: int, T: int) -> bool:
    """Whether T rows of y (N values at yp, stride ldy) and x share memory;
    column ranges of one buffer do not, though their address ranges cross."""
    ye, xe = (2 if ycode else 4), (2 if xcode else 4)
    yl, xl, yw, xw = ldy * ye, ldx * xe, N * ye, K * xe
    if yp >= xp + (T - 1) * xl + xw or xp >= yp + (T - 1) * yl + yw:
        return False
    if T <= 1 or yl != xl:
        return True
    d = (xp - yp) % yl  # x's columns start d bytes behind y's in a row of the buffer
    return d < yw or d + xw > yl


def is_host(a) -> bool:
    return not (isinstance(a, torch.Tensor) and a.is_cuda)


def to_device(a, dtype: torch.dtype | None = None) -> torch.Tensor:
    """numpy / bytes / torch -> contiguous tensor on the current GPU."""
    if (isinstance(a, torch.Tensor) and a.is_cuda and (dtype is None or a.dtype == dtype) and a.is_contiguous()
            and a.get_device() == torch.cuda.current_device()):
        return a  # what the conversions below return for it, without their 1.9 us
    dev = require_gpu()
    if isinstance(a, (bytes, bytearray, memoryview)):
        a = np.frombuffer(a, dtype=np.uint8)
    if isinstance(a, np.ndarray):
        with warnings.catch_warnings():
            # read-only arrays (np.frombuffer over weight bytes) are only read here: uploaded, never written
            warnings.filterwarnings("ignore", message="The given NumPy array is not writable")
            t = torch.from_numpy(np.ascontiguousarray(a))
    elif isinstance(a, torch.Tensor):
        t = a
    else:
        t = torch.as_tensor(a)
    if dtype is not None and t.dtype != dtype:
        t = t.to(dtype)
    return t.to(dev, non_blocking=False).contiguous()


def half_for_mfma(x_f32: torch.Tensor, host=None) -> torch.dtype:
    """The 16-bit type float32 activations take into a bf16 / fp16 MFMA:
    float16 (11 significant bits) when every |x| is finite and fits its
    range, else bfloat16 (8 bits, float32's range).  ``host``: the same
    values as a host array, when the caller has them (no device read)."""
    if x_f32.numel() == 0:
        amax = 0.0
    elif host is not None:
        amax = float(np.abs(np.asarray(host, np.float32)).max())
    else:
        amax = float(x_f32.abs().amax().item())
    return torch.float16 if np.isfinite(amax) and amax <= 65504.0 else torch.bfloat16


def to_host(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().numpy()


def raw_u8(weight_bytes) -> torch.Tensor:
    """The reference passes weights as raw bytes or any ndarray (reinterpreted
    as uint8, ``quant/method.py:103-106``); return a uint8 device view."""
    if isinstance(weight_bytes, torch.Tensor):
        t = weight_bytes if weight_bytes.is_cuda else to_device(weight_bytes)
        return t.contiguous().view(torch.uint8).reshape(-1)
    if isinstance(weight_bytes, (bytes, bytearray, memoryview)):
        return to_device(np.frombuffer(weight_bytes, dtype=np.uint8))
    arr = np.ascontiguousarray(np.asarray(weight_bytes))
    return to_device(arr.reshape(-1).view(np.uint8))


_WS: dict[tuple, torch.Tensor] = {}


def workspace(tag: str, nbytes: int, device: torch.device | None = None) -> torch.Tensor:
    """Per-device, per-tag zero-initialised scratch that only grows.  Kernels
    that use counters in it leave them at zero after every call, so the buffer
    is zeroed only when (re)allocated."""
    dev = device or require_gpu()
    key = (tag, dev.index)
    buf = _WS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=dev)
        _WS[key] = buf
    return buf
