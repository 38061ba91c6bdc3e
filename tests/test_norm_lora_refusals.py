"""ccq_rms_norm, ccq_lora_add and ccq_fp8_block_linear_quantized refuse bad
arguments on the host before anything is launched, and the Python entry points
refuse host tensors (runs without a GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)  # never dereferenced: validation comes first


@pytest.fixture(scope="module")
def lib(built_lib):
    from ccut import _lib

    return _lib.lib()


def _norm(lib, **kw):
    a = dict(x=P, x_dtype=2, ldx=256, residual=None, ldr=0, w=P, w_dtype=2, eps=1e-6, residual_out=None, ldo=0, y=None,
             y_dtype=0, q_fmt=1, q=P, scale=P, rows=2, H=256)
    a.update(kw)
    return lib.ccq_rms_norm(*a.values(), None)


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(H=0), "H="), (dict(H=32769, ldx=32769, q_fmt=2), "H="),
    (dict(H=200), "multiple of 128"), (dict(x_dtype=3), "x_dtype"), (dict(w_dtype=-1), "w_dtype"),
    (dict(y=P, y_dtype=9), "y_dtype"), (dict(q_fmt=3), "q_fmt"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(ldx=255), "stride"), (dict(residual=P, ldr=255), "stride"),
    (dict(residual_out=P, ldo=0), "stride"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(q=None), "null"),
    (dict(scale=None), "null"), (dict(q_fmt=0, q=None, scale=None), "null"), (dict(x=ctypes.c_void_p(257)), "aligned"),
    (dict(w_dtype=0, w=ctypes.c_void_p(258)), "aligned"), (dict(q=ctypes.c_void_p(260)), "8-byte"),
])
def test_rms_norm(lib, kw, word):
    from ccut._lib import CCQ_EINVAL, last_error

    assert _norm(lib, **kw) == CCQ_EINVAL and word in last_error()


def test_empty_calls(lib):
    from ccut._lib import ccq_lora_adapters

    assert _norm(lib, rows=0) == 0
    ad = ccq_lora_adapters(256, 256, None, None, 2, 3, 16, 64, 48)
    assert lib.ccq_lora_add(P, 2, 64, P, P, 2, 48, 0, ad, None, 0, None) == 0
    assert lib.ccq_lora_workspace_size(P, 2, 64, 0, ad) == 0
    assert lib.ccq_fp8_block_linear_quantized(P, P, P, P, P, 2, 0, 256, 128, None) == 0


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=0), "f16 or bf16"), (dict(L=0), "num_adapters"), (dict(L=1025), "num_adapters"), (dict(R=0), "rank_max"),
    (dict(R=257), "rank_max"), (dict(K=0), "in_features"), (dict(N=(1 << 20) + 1), "out_features"), (dict(T=-1), "T="),
    (dict(T=65537), "T="), (dict(x_dtype=3), "x_dtype"), (dict(y_dtype=-2), "y_dtype"), (dict(ldx=63), "stride"),
    (dict(ldy=47), "stride"), (dict(a=None), "null"), (dict(b=None), "null"), (dict(x=None), "null"),
    (dict(index=None), "null"), (dict(y=None), "null"), (dict(x=ctypes.c_void_p(257)), "aligned"),
    (dict(index=ctypes.c_void_p(260)), "aligned"), (dict(ws=None), "workspace"), (dict(ws_bytes=16), "workspace"),
    (dict(ws=ctypes.c_void_p(264)), "workspace"),
])
def test_lora(lib, kw, word):
    from ccut._lib import CCQ_EINVAL, ccq_lora_adapters, last_error

    a = dict(x=P, x_dtype=2, ldx=64, index=P, y=P, y_dtype=2, ldy=48, T=600, ws=P, ws_bytes=1 << 30, a=256, b=256, dtype=2,
             L=3, R=16, K=64, N=48)
    a.update(kw)
    ad = ccq_lora_adapters(a["a"], a["b"], None, None, a["dtype"], a["L"], a["R"], a["K"], a["N"])
    rc = lib.ccq_lora_add(a["x"], a["x_dtype"], a["ldx"], a["index"], a["y"], a["y_dtype"], a["ldy"], a["T"], ad, a["ws"],
                          a["ws_bytes"], None)
    assert rc == CCQ_EINVAL and word in last_error()


@pytest.mark.parametrize("args,word", [
    ((P, P, P, P, P, 2, -1, 256, 128), "negative"), ((P, P, P, P, P, 2, 4, 200, 128), "128"),
    ((P, P, P, P, P, 2, 4, 256, 100), "128"), ((P, P, P, P, P, 2, 4, 128, 128), "256"),
    ((P, P, P, P, P, 7, 4, 256, 128), "y_dtype"), ((None, P, P, P, P, 2, 4, 256, 128), "null"),
    ((P, None, P, P, P, 2, 4, 256, 128), "null"), ((P, P, None, P, P, 2, 4, 256, 128), "null"),
    ((ctypes.c_void_p(264), P, P, P, P, 2, 4, 256, 128), "aligned"),
    ((P, P, P, P, P, 2, 1 << 25, 256, 128), "4 GiB"),
])
def test_fp8_linear_quantized(lib, args, word):
    from ccut._lib import CCQ_EINVAL, last_error

    assert lib.ccq_fp8_block_linear_quantized(*args, None) == CCQ_EINVAL and word in last_error()


def test_host_tensors():
    from ccut.blocks import norm
    from ccut.quant import fp8_block, lora

    x = torch.zeros((2, 256), dtype=torch.bfloat16)
    for f in (norm.rms_norm_fp8, norm.rms_norm_int8):
        with pytest.raises(ValueError, match="cpu"):
            f(x, x[0])
    with pytest.raises(ValueError, match="cpu"):
        lora.LoraAdapters(torch.zeros((1, 8, 256), dtype=torch.bfloat16), torch.zeros((1, 64, 8), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="cpu"):
        lora.add_(torch.zeros((2, 64)), x, None, torch.zeros(2, dtype=torch.int64))
    w = fp8_block.Fp8BlockWeights(torch.zeros(128 * 256, dtype=torch.uint8), torch.zeros((1, 2)), 128, 256)
    with pytest.raises(ValueError, match="cpu"):
        fp8_block.linear_quantized(w, x.to(torch.uint8), torch.zeros((2, 2)))


def test_overlap_of_views():
    """Which views of one buffer count as overlapping."""
    from ccut import _dev
    from ccut.quant import lora

    def over(y, x):
        return lora._overlap(y.data_ptr(), _dev.DTYPE_CODE[y.dtype], y.stride(0), y.shape[1], x.data_ptr(),
                             _dev.DTYPE_CODE[x.dtype], x.stride(0), x.shape[1], y.shape[0])

    buf = torch.zeros((6, 100))
    assert not over(buf[:, :40], buf[:, 40:])
    assert not over(buf[:, 60:], buf[:, :60])
    assert over(buf[:, :41], buf[:, 40:])
    assert over(buf[:, 30:70], buf[:, :31])
    assert over(buf, buf)
    assert not over(buf[:3], buf[3:])
    assert over(buf[:3], buf[2:5])
    assert not over(buf[1:4, 50:], buf[2:5, :50])
    assert over(buf[:1, :40], buf[:1, 39:])
    assert not over(torch.zeros((6, 40)), torch.zeros((6, 40)))
    half = buf.view(torch.float16)  # 200 columns of half the size
    assert not over(half[:, :80], buf[:, 40:])
    assert over(half[:, :81], buf[:, 40:])


def test_rms_norm_packed(lib):
    """The arguments in one block reach the same checks, each from its place."""
    from ccut._lib import CCQ_EINVAL, RMS_NORM_ARGS, last_error

    def call(**kw):
        a = dict(x=256, residual=0, w=256, residual_out=0, y=0, q=256, scale=256, stream=0, ldx=256, ldr=0, ldo=0, rows=2,
                 H=256, x_dtype=2, w_dtype=2, y_dtype=0, q_fmt=1, eps=1e-6)
        a.update(kw)
        return lib.ccq_rms_norm_packed(RMS_NORM_ARGS.pack(*a.values()))

    assert RMS_NORM_ARGS.size == 128
    assert call(rows=0) == 0
    for kw, word in [(dict(rows=-1), "rows"), (dict(H=200), "multiple of 128"), (dict(x_dtype=3), "x_dtype"),
                     (dict(w_dtype=-1), "w_dtype"), (dict(y=256, y_dtype=9), "y_dtype"), (dict(q_fmt=3), "q_fmt"),
                     (dict(eps=0.0), "eps"), (dict(ldx=255), "stride"), (dict(residual=256, ldr=255), "stride"),
                     (dict(residual_out=256, ldo=0), "stride"), (dict(x=0), "null"), (dict(w=0), "null"),
                     (dict(q=0), "null"), (dict(scale=0), "null"), (dict(x=257), "aligned"), (dict(q=260), "8-byte")]:
        assert call(**kw) == CCQ_EINVAL and word in last_error(), kw
    assert lib.ccq_rms_norm_packed(None) == CCQ_EINVAL and "null" in last_error()


def test_without_torch_internals():
    """A torch that lacks the internal short cuts (one built for the CPU, or
    another release) still imports the package, on which host-only code
    stands, and allocates by the public calls."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
del torch._C._dynamo.guards._empty_strided_cuda
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import ccut.blocks.norm, ccut.quant.lora, ccut.quant.registry
from ccut import _dev
made = []
torch.empty_strided = lambda *a, **k: made.append((a, k))
_dev.empty_strided((2, 3), (3, 1), torch.float32)
assert made == [(((2, 3), (3, 1)), dict(dtype=torch.float32, device="cuda"))], made
torch.cuda.current_device = lambda: 5
assert _dev.is_current(5) and not _dev.is_current(0)
torch.cuda.current_stream = lambda device: type("S", (), dict(cuda_stream=100 + device))
assert _dev.raw_stream(3) == 103 and _dev.stream_ptr(torch.device("cuda", 2)) == 102
print("ok")
"""
    pkg = Path(__file__).resolve().parents[1] / "costcut-infer_amd"
    r = subprocess.run([sys.executable, "-c", code, str(pkg)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stderr[-2000:]
