"""RMS norm with the residual's addition and 8-bit rows (``ccq_rms_norm``)
against a plain computation: codes and residual bit by bit (they are exact
functions of the float32 products), scales and normalized rows to the rounding
of the row's float32 statistics."""

from __future__ import annotations

import pytest
import torch

from oracle import norm as on

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
# mean(s^2): at most 32 fused adds per thread, 6 steps in a wave, 16 waves, the division and eps (56 roundings, half
# of them left by the square root); sqrt, reciprocal, and the two of scale or y
REL = (56 / 2 + 4) * U
EPS = 1e-6


def _close(got, ref, dtype=torch.float32):
    got, ref = got.cpu().double(), ref.double()
    assert torch.equal(got.isnan(), ref.isnan())
    ok = ~ref.isnan()
    eps = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tol = ref.abs() * (REL + eps) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = (got - ref).abs() > tol
    assert not bad[ok].any(), f"worst {((got - ref).abs() / ref.abs().clamp_min(1e-30))[ok].max():.3e}"


def _case(T, H, dt, residual, seed=0, wdt=None):
    g = torch.Generator().manual_seed(seed * 1000003 + T * 31 + H)
    x = torch.randn((T, H), generator=g).to(dt)
    r = (torch.randn((T, H), generator=g) * torch.exp(torch.randn(H, generator=g))).to(dt) if residual else None
    w = (1 + 0.2 * torch.randn(H, generator=g)).to(wdt or dt)
    return x, w, r


def _check(got, x, w, r, fmt, normed, eps=EPS):
    s, p, rstd, y = on.rms_norm(x, w, eps, r)
    q, scale = on.fp8_rows(p, rstd) if fmt == "fp8" else on.int8_rows(p, rstd)
    assert torch.equal(got.q.cpu(), q)
    _close(got.scale, scale)
    assert (got.y is not None) == normed and (got.residual is not None) == (r is not None)
    if normed:
        _close(got.y, y, x.dtype)
    if r is not None:
        assert torch.equal(got.residual.cpu(), s.to(x.dtype))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H", [1, 7, 8, 130, 511, 512, 513, 2048, 2049, 4095, 4096, 4097, 8192, 8195, 32768])
def test_int8_rows(gpu, H, dt):
    from ccut.blocks import norm

    for T, residual, normed in ((1, True, False), (6, False, True), (9, True, True)):
        x, w, r = _case(T, H, DT[dt], residual)
        got = norm.rms_norm_int8(x.to(gpu), w.to(gpu), EPS, residual=None if r is None else r.to(gpu), normed=normed)
        _check(got, x, w, r, "int8", normed)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H", [128, 256, 384, 512, 640, 2048, 2176, 4096, 5632, 7168, 8192, 8320, 32768])
def test_fp8_rows(gpu, H, dt):
    from ccut.blocks import norm

    for T, residual, normed in ((1, True, False), (5, False, True), (67, True, True)):
        x, w, r = _case(T, H, DT[dt], residual)
        got = norm.rms_norm_fp8(x.to(gpu), w.to(gpu), EPS, residual=None if r is None else r.to(gpu), normed=normed)
        _check(got, x, w, r, "fp8", normed)


@pytest.mark.parametrize("wdt", ["bf16", "f16", "f32"])
def test_weight_types_and_plain_rows(gpu, wdt):
    from ccut.blocks import norm

    for H in (100, 2048, 4100):
        x, w, r = _case(33, H, torch.bfloat16, True, wdt=DT[wdt])
        s, _, _, y = on.rms_norm(x, w, EPS, r)
        got, res = norm.rms_norm(x.to(gpu), w.to(gpu), EPS, residual=r.to(gpu))
        _close(got, y, torch.bfloat16)
        assert torch.equal(res.cpu(), s.bfloat16())
        y0 = on.rms_norm(x, w, EPS)[3]
        _close(norm.rms_norm(x.to(gpu), w.to(gpu), EPS, out_dtype=torch.float32), y0)
        _close(norm.rms_norm(x.to(gpu), w.to(gpu), EPS, out_dtype=torch.float16), y0, torch.float16)
        # host rows in, host rows out
        yn, rn = norm.rms_norm(x.float().numpy(), w.float().numpy(), EPS, residual=r.float().numpy())
        _close(torch.from_numpy(yn), y)
        assert torch.equal(torch.from_numpy(rn), s)


def test_shapes_strides_and_alignment(gpu):
    """Leading dimensions, columns of a larger buffer at odd offsets, no rows,
    and rows that the call must not touch."""
    from ccut.blocks import norm

    for H, off in ((128, 1), (384, 3), (2176, 5)):
        x, w, r = _case(12, H, torch.bfloat16, True)
        big = torch.full((14, 2 * H + 9), 7.0, dtype=torch.bfloat16, device=gpu)
        xs, rs = big[1:13, off:off + H], big[1:13, off + H:off + 2 * H]
        xs.copy_(x.to(gpu))
        rs.copy_(r.to(gpu))
        before = big.clone()
        got = norm.rms_norm_fp8(xs, w.to(gpu), EPS, residual=rs, normed=True)
        _check(got, x, w, r, "fp8", True)
        assert torch.equal(big, before)
        got = norm.rms_norm_int8(xs, w.to(gpu), EPS, residual=rs, residual_out=rs)
        _check(got, x, w, r, "int8", False)
        assert got.residual.data_ptr() == rs.data_ptr()
        before[1:13, off + H:off + 2 * H] = on.rms_norm(x, w, EPS, r)[0].bfloat16().to(gpu)
        assert torch.equal(big, before)
        # the sum written over x
        rs.copy_(r.to(gpu))
        got = norm.rms_norm_int8(xs, w.to(gpu), EPS, residual=rs, residual_out=xs)
        _check(got, x, w, r, "int8", False)
        assert torch.equal(xs.cpu(), on.rms_norm(x, w, EPS, r)[0].bfloat16())
    x, w, r = _case(12, 256, torch.float16, True)
    shaped = [t.reshape(2, 3, 2, 256) for t in (x, r)]
    got = norm.rms_norm_fp8(shaped[0].to(gpu), w.to(gpu), EPS, residual=shaped[1].to(gpu), normed=True)
    assert got.q.shape == (2, 3, 2, 256) and got.scale.shape == (2, 3, 2, 2) and got.y.shape == (2, 3, 2, 256)
    _check(got, shaped[0], w, shaped[1], "fp8", True)
    one = norm.rms_norm_int8(x[0].to(gpu), w.to(gpu), EPS)
    assert one.q.shape == (256,) and one.scale.shape == ()
    _check(one, x[0], w, None, "int8", False)
    turned = torch.randn(256, 5, device=gpu).t()  # rows that are columns
    _check(norm.rms_norm_int8(turned, w.to(gpu), EPS), turned.cpu(), w, None, "int8", False)
    none = norm.rms_norm_fp8(torch.empty((0, 256), dtype=torch.float16, device=gpu), w.to(gpu), normed=True)
    assert none.q.shape == (0, 256) and none.scale.shape == (0, 2) and none.y.shape == (0, 256)


def test_special_rows(gpu):
    """Zero rows, NaN, infinities, very small and very large values."""
    from ccut.blocks import norm

    for H in (256, 1024, 8320):
        x, w, _ = _case(9, H, torch.float32, False)
        x[1] = 0.0
        x[2, 5] = float("nan")
        x[3, 200] = float("inf")
        x[4] *= 1e-18
        x[5] *= 1e15
        x[6, :128] = 0.0           # one block of zeros
        x[7] = -0.0
        x[8] *= 1e-33              # products below the smallest divisor of a code
        f8 = norm.rms_norm_fp8(x.to(gpu), w.to(gpu), EPS, normed=True)
        i8 = norm.rms_norm_int8(x.to(gpu), w.to(gpu), EPS, normed=True)
        finite = [0, 1, 4, 5, 6, 7, 8]
        s, p, rstd, y = on.rms_norm(x, w, EPS)
        for got, rows in ((f8, on.fp8_rows), (i8, on.int8_rows)):
            q, scale = rows(p, rstd)
            assert torch.equal(got.q.cpu()[finite], q[finite])
            _close(got.scale[finite], scale[finite])
            _close(got.y[finite], y[finite])
            assert got.scale[2].isnan().all() and got.y[2].isnan().all()
            # an infinity: rstd is 0, so 0 elsewhere and NaN at it
            assert torch.equal(got.y[3].isnan().cpu(), torch.arange(H) == 200)
            assert (got.y[3].nan_to_num() == 0).all()
        deq = f8.q[3].view(torch.float8_e4m3fn).float().view(-1, 128) * f8.scale[3][:, None]
        assert deq[1].isnan().any() and (deq[torch.arange(H // 128) != 1] == 0).all()
        assert i8.scale[3].isnan()


def test_captured_and_two_streams(gpu):
    """A captured call replays on new rows like the eager one, with eager work
    between the replays; two streams at once give what one gives."""
    from ccut.blocks import norm

    T, H = 70, 2176
    cases = [tuple(t.to(gpu) for t in _case(T, H, torch.bfloat16, True, seed=s)) for s in range(4)]
    x, w, r = (t.clone() for t in cases[0])
    norm.rms_norm_fp8(x, w, EPS, residual=r, normed=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = norm.rms_norm_fp8(x, w, EPS, residual=r, normed=True)
    eager = [norm.rms_norm_fp8(*c[:2], EPS, residual=c[2], normed=True) for c in cases]
    for n in (1, 2, 3, 0):
        x.copy_(cases[n][0])
        w.copy_(cases[n][1])
        r.copy_(cases[n][2])
        graph.replay()
        again = norm.rms_norm_fp8(*cases[n][:2], EPS, residual=cases[n][2], normed=True)
        torch.cuda.synchronize()
        for a, b, c in zip(held, eager[n], again):
            assert torch.equal(a, b) and torch.equal(b, c)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for n, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got[n] = norm.rms_norm_fp8(*cases[n][:2], EPS, residual=cases[n][2], normed=True)
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[n], eager[n]))


def test_far_rows(gpu):
    """Row offsets beyond 2^31 elements."""
    from ccut.blocks import norm

    T, H, ld = 40000, 128, 65536
    buf = torch.empty((T, ld), dtype=torch.bfloat16, device=gpu)
    x = buf[:, 17:17 + H]
    x.copy_(torch.randn((T, H), generator=torch.Generator(device=gpu).manual_seed(1), device=gpu))
    w = torch.ones(H, device=gpu)
    got = norm.rms_norm_fp8(x, w, EPS)
    dense = norm.rms_norm_fp8(x.contiguous(), w, EPS)
    assert torch.equal(got.q, dense.q) and torch.equal(got.scale, dense.scale)
    tail = slice(T - 50, T)
    _check(norm.QuantizedRows(got.q[tail], got.scale[tail], None, None), x[tail].cpu(), w.cpu(), None, "fp8", False)


def test_refusals(gpu):
    from ccut.blocks import norm

    x, w = torch.zeros((3, 256), device=gpu), torch.ones(256, device=gpu)
    bad = [
        lambda: norm.rms_norm_fp8(torch.zeros((3, 200), device=gpu), torch.ones(200, device=gpu)),
        lambda: norm.rms_norm_fp8(x, w[:255]),
        lambda: norm.rms_norm_fp8(x, w.cpu()),
        lambda: norm.rms_norm_fp8(x.double(), w),
        lambda: norm.rms_norm_fp8(x, w.double()),
        lambda: norm.rms_norm_fp8(x, w, 0.0),
        lambda: norm.rms_norm_fp8(x, w, float("nan")),
        lambda: norm.rms_norm_fp8(x, w, float("inf")),
        lambda: norm.rms_norm_fp8(x, w, residual=x[:2]),
        lambda: norm.rms_norm_fp8(x, w, residual=x.half()),
        lambda: norm.rms_norm_fp8(x, w, residual=x.cpu()),
        lambda: norm.rms_norm_fp8(x, w, residual_out=x),
        lambda: norm.rms_norm_fp8(x, w, residual=x, residual_out=torch.zeros((256, 3), device=gpu).t()),
        lambda: norm.rms_norm_fp8(x, w, residual=x, residual_out=torch.zeros(256, device=gpu).expand(3, 256)),
        lambda: norm.rms_norm_int8(torch.zeros((3, 0), device=gpu), torch.zeros(0, device=gpu)),
        lambda: norm.rms_norm_int8(torch.zeros((1, 32769), device=gpu), torch.zeros(32769, device=gpu)),
        lambda: norm.rms_norm(x, w, out_dtype=torch.float64),
        lambda: norm.rms_norm(x.cpu().numpy(), w.cpu().numpy(), residual=x, residual_out=x),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print(f"call {i} was not refused")


def test_very_many_rows(gpu):
    """More rows than one launch takes."""
    from ccut.blocks import norm

    for T, H in ((2 ** 23 + 1037, 2), (2 ** 21 + 37, 520)):
        x = torch.randn((T, H), generator=torch.Generator(device=gpu).manual_seed(H), device=gpu).bfloat16()
        w = torch.linspace(0.5, 1.5, H, device=gpu)
        got = norm.rms_norm_int8(x, w, EPS, normed=True)
        for t in range(0, T, 2 ** 20):
            part = norm.rms_norm_int8(x[t:t + 2 ** 20], w, EPS, normed=True)
            assert all(torch.equal(a[t:t + 2 ** 20], b) for a, b in zip(got[:3], part[:3])), f"rows from {t}"
        tail = slice(T - 40, T)
        _check(norm.QuantizedRows(*(t[tail] for t in got[:3]), None), x[tail].cpu(), w.cpu(), None, "int8", True)

    T, H = 2 ** 21 + 37, 128  # FP8, strided rows, the sum in place
    buf = torch.randn((T, 2 * H + 8), generator=torch.Generator(device=gpu).manual_seed(1), device=gpu).half()
    x, res = buf[:, :H], buf[:, H:2 * H]
    before, w = res.clone(), torch.linspace(0.5, 1.5, H, device=gpu)
    got = norm.rms_norm_fp8(x, w, EPS, residual=res, residual_out=res, normed=True)
    for rows in (slice(0, 50), slice(2 ** 21 - 20, T)):
        part = norm.QuantizedRows(*(t[rows] for t in got))
        _check(part, x[rows].cpu(), w.cpu(), before[rows].cpu(), "fp8", True)


def test_sum_over_another_view_is_refused(gpu):
    from ccut.blocks import norm

    buf, w = torch.zeros((8, 512), device=gpu), torch.ones(256, device=gpu)
    x, r = buf[:4, :256], torch.zeros((4, 256), device=gpu)
    for out in (buf[1:5, :256], buf[:4, 1:257], buf[:4].view(8, 256)[:4]):
        for a, b in ((x, r), (r, x)):
            with pytest.raises(ValueError, match="overlaps"):
                norm.rms_norm_int8(a, w, residual=b, residual_out=out)
    for out in (buf[:4, 256:], buf[4:, :256], x, r):
        assert norm.rms_norm_int8(x, w, residual=r, residual_out=out).residual is out


def test_public_allocation_and_stream_calls(gpu, monkeypatch):
    """The calls that stand in for torch's internal short cuts give the same
    rows, on a stream of their own too."""
    from ccut import _dev
    from ccut.blocks import norm

    x, w, r = (t.to(gpu) for t in _case(9, 256, torch.bfloat16, True))
    want = norm.rms_norm_fp8(x, w, EPS, residual=r, normed=True)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        assert _dev._raw_stream(0) == _dev.raw_stream(0) == st.cuda_stream
        monkeypatch.setattr(norm, "empty_strided", _dev._empty_strided)
        monkeypatch.setattr(norm, "raw_stream", _dev._raw_stream)
        monkeypatch.setattr(_dev, "current_device", _dev._current_device)
        got = norm.rms_norm_fp8(x, w, EPS, residual=r, normed=True)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_host_rows_are_returned_as_float32(gpu):
    """Another type for host rows is refused, not left out."""
    from ccut.blocks import norm

    x, w = torch.randn(3, 40), torch.ones(40)
    y = norm.rms_norm(x.numpy(), w.numpy(), EPS, out_dtype=torch.float32)
    assert y.dtype.name == "float32"
    _close(torch.from_numpy(y), on.rms_norm(x, w, EPS)[3])
    for dt in (torch.float16, torch.bfloat16, torch.float64):
        with pytest.raises(ValueError, match="float32"):
            norm.rms_norm(x.numpy(), w.numpy(), EPS, out_dtype=dt)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H", [2049, 2176, 4095, 4096, 4097, 7168, 8191, 8192])
def test_both_sides_of_the_row_count_rule(gpu, H, dt):
    """More than 512 rows take two vectors a thread, fewer one, for rows of
    2049 to 8192: every output format on both."""
    from ccut.blocks import norm

    for T in (512, 513, 530):
        x, w, r = _case(T, H, DT[dt], T != 513)
        xd, wd, rd = x.to(gpu), w.to(gpu), None if r is None else r.to(gpu)
        _check(norm.rms_norm_int8(xd, wd, EPS, residual=rd, normed=True), x, w, r, "int8", True)
        if H % 128 == 0:
            _check(norm.rms_norm_fp8(xd, wd, EPS, residual=rd, normed=True), x, w, r, "fp8", True)
        y = on.rms_norm(x, w, EPS, r)[3]
        got = norm.rms_norm(xd, wd, EPS, residual=rd)
        _close(got if r is None else got[0], y, x.dtype)


@pytest.mark.parametrize("H", [9000, 16384, 16385, 20000])
def test_long_rows(gpu, H):
    """The two instances above 8192 columns, few rows and many."""
    from ccut.blocks import norm

    for T, dt in ((3, "f32"), (600, "bf16"), (40, "f16")):
        x, w, r = _case(T, H, DT[dt], True)
        xd, wd, rd = x.to(gpu), w.to(gpu), r.to(gpu)
        _check(norm.rms_norm_int8(xd, wd, EPS, residual=rd, normed=True), x, w, r, "int8", True)
        if H % 128 == 0:
            _check(norm.rms_norm_fp8(xd, wd, EPS, residual=rd, normed=True), x, w, r, "fp8", True)


def test_rows_whose_squares_overflow(gpu):
    """Finite values whose squares leave float32: the row's statistics are
    infinite, so y and the scales are 0, with the codes as defined."""
    from ccut.blocks import norm

    x, w, _ = _case(4, 1024, torch.float32, False)
    x[1] *= 1e25
    x[2, 700] = 1e30
    for f, rows in ((norm.rms_norm_fp8, on.fp8_rows), (norm.rms_norm_int8, on.int8_rows)):
        got = f(x.to(gpu), w.to(gpu), EPS, normed=True)
        _, p, rstd, y = on.rms_norm(x, w, EPS)
        q, scale = rows(p, rstd)
        assert torch.equal(got.q.cpu(), q)
        for t in (1, 2):
            assert (got.scale[t] == 0).all() and (got.y[t] == 0).all()
        for t in (0, 3):
            _close(got.scale[t], scale[t])
            _close(got.y[t], y[t])
