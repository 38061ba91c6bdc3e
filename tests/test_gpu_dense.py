"""Linears with 16-bit weights and an epilogue (``ccq_dense_linear``,
``ccq_dense_linear_grouped``) against the 64-bit product, element by element
within the bound that float32 sums, the activation's evaluation and y's
rounding allow (``oracle.dense``)."""

from __future__ import annotations

import pytest
import torch

from oracle import dense as od
from oracle import permute as op

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPILOGUES = [(False, None, None, False), (True, "silu", F32, False), (False, "gelu", "same", True),
             (False, "gelu_tanh", None, True), (True, "relu", "same", True), (True, None, None, False),
             (True, "gelu", BF, False), (True, "gelu_tanh", F16, True)]


def _inputs(M, K, N, dt, gated, bias, residual, ydt, seed=0, E=None):
    g = torch.Generator().manual_seed(seed * 7919 + M * 131 + K * 17 + N * 3)
    W = 2 * N if gated else N
    lead = () if E is None else (E,)
    c = dict(x=torch.randn((M, K), generator=g).to(dt), w=(torch.randn((*lead, W, K), generator=g) * K ** -0.5).to(dt),
             bias=None, residual=None)
    if bias is not None:
        c["bias"] = torch.randn((*lead, W), generator=g).to(dt if bias == "same" else bias)
    if residual:
        c["residual"] = (torch.randn((M, N), generator=g) * 2).to(ydt)
    return c


def _up(t, gpu):
    return None if t is None else t.to(gpu)


def _close(y, ref, bound, what=""):
    assert torch.isfinite(y).all()
    off, tol = (y.cpu().double() - ref).abs(), bound(y.dtype)
    assert (off <= tol).all(), f"{what} worst {(off / tol).max():.3f} of the bound"


def _run(gpu, c, gated, act, ydt=None, **kw):
    from ccut.quant import dense

    y = dense.linear(_up(c["x"], gpu), _up(c["w"], gpu), _up(c["bias"], gpu), act=act, gated=gated,
                     residual=_up(c["residual"], gpu), out_dtype=ydt, **kw)
    ref, bound = od.linear(c["x"], c["w"], c["bias"], act, gated, c["residual"])
    _close(y, ref, bound)
    return y


@pytest.mark.parametrize("gated,act,bias,residual", EPILOGUES)
@pytest.mark.parametrize("dt,ydt", [(BF, BF), (F16, F16), (BF, F32), (F16, BF)])
@pytest.mark.parametrize("M,K,N", [(1, 256, 320), (16, 512, 96), (17, 100, 33), (93, 205, 147), (300, 384, 264)])
def test_epilogues(gpu, M, K, N, dt, ydt, gated, act, bias, residual):
    _run(gpu, _inputs(M, K, N, dt, gated, bias, residual, ydt), gated, act, ydt)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 600])
def test_rows(gpu, M):
    for dt, gated in ((BF, False), (F16, True)):
        _run(gpu, _inputs(M, 192, 160, dt, gated, None, True, dt), gated, "silu")


@pytest.mark.parametrize("K", [1, 2, 7, 8, 9, 31, 33, 63, 64, 65, 72, 127, 128, 136, 513, 1024, 1031, 4096, 14336])
def test_inner_sizes(gpu, K):
    for M, dt in ((1, BF), (20, F16), (50, BF), (70, F16), (270, BF)):
        _run(gpu, _inputs(M, K, 80, dt, False, "same", False, dt), False, None)


@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 15, 16, 17, 31, 33, 63, 65, 127, 129, 130, 255, 257, 1000])
def test_outer_sizes(gpu, N):
    for M, dt, gated in ((1, BF, True), (40, F16, False), (70, BF, True), (260, F16, False)):
        _run(gpu, _inputs(M, 136, N, dt, gated, F32, True, dt), gated, "gelu")


@pytest.mark.parametrize("M,K,N", [(2048, 192, 6200), (2050, 264, 6272), (1000, 328, 12416)])
@pytest.mark.parametrize("gated", [False, True])
def test_many_tiles(gpu, M, K, N, gated):
    c = _inputs(M, K, N // 2 if gated else N, BF, gated, F32, True, BF)
    _run(gpu, c, gated, "silu" if gated else None)


@pytest.mark.parametrize("M,K,N", [(65, 8192, 64), (128, 14336, 128), (93, 4097, 131), (200, 5000, 300), (135, 6664, 5524)])
def test_long_inner(gpu, M, K, N):
    for gated, dt in ((False, BF), (True, F16)):
        _run(gpu, _inputs(M, K, N, dt, gated, "same", True, dt), gated, "relu")


@pytest.mark.parametrize("M", [3, 90, 300])
def test_strides_and_alignment(gpu, M):
    """Rows cut out of wider buffers, at addresses of every alignment."""
    from ccut.quant import dense

    K, N = 136, 72
    for shift in range(0, 9):
        for pad in (0, 1, 5, 8):
            c = _inputs(M, K, N, BF, False, "same", True, BF, seed=shift * 16 + pad)
            x, r, o = (torch.full((M * (w + pad) + 32,), 7.0, dtype=BF, device=gpu) for w in (K, N, N))
            view = lambda t, w: t[shift:shift + M * (w + pad)].view(M, w + pad)[:, :w]  # noqa: E731
            view(x, K).copy_(c["x"])
            view(r, N).copy_(c["residual"])
            out = view(o, N)
            y = dense.linear(view(x, K), c["w"].to(gpu), c["bias"].to(gpu), act="gelu", residual=view(r, N), out=out)
            assert y is out
            ref, bound = od.linear(c["x"], c["w"], c["bias"], "gelu", False, c["residual"])
            _close(y, ref, bound)
            rest = torch.ones_like(o, dtype=torch.bool)
            view(rest, N).fill_(False)
            assert (o[rest] == 7.0).all()


@pytest.mark.parametrize("M", [1, 5, 16, 40])
@pytest.mark.parametrize("K", [7, 31, 257, 511, 1024, 2049])
def test_odd_elements(gpu, M, K):
    """Rows of x and w that start at odd and even elements, NaN around them."""
    from ccut.quant import dense

    N = 70
    for shift, pad in ((0, 0), (1, 0), (0, 1), (1, 2), (3, 1), (2, 0)):
        c = _inputs(M, K, N, BF, False, None, False, BF, seed=shift)
        x = torch.full((M * (K + pad) + 16,), float("nan"), dtype=BF, device=gpu)[shift:shift + M * (K + pad)]
        x = x.view(M, K + pad)[:, :K].copy_(c["x"])
        w = torch.full((N * K + 16,), float("nan"), dtype=BF, device=gpu)[3 - shift:3 - shift + N * K].view(N, K)
        w.copy_(c["w"])
        ref, bound = od.linear(c["x"], c["w"])
        _close(dense.linear(x, w), ref, bound)
        if M > 1:
            offsets = torch.tensor([0, M // 2, M], dtype=torch.int32, device=gpu)
            y = dense.linear_grouped(x, offsets, w.view(2, N // 2, K))
            left, right = od.linear(c["x"][:M // 2], c["w"][:N // 2]), od.linear(c["x"][M // 2:], c["w"][N // 2:])
            _close(y[:M // 2], *left)
            _close(y[M // 2:], *right)


def test_transposed_and_leading_dimensions(gpu):
    from ccut.quant import dense

    c = _inputs(30, 64, 48, BF, False, "same", True, BF)
    ref, bound = od.linear(c["x"], c["w"], c["bias"], "silu", False, c["residual"])
    x = c["x"].to(gpu).t().contiguous().t()          # rows not dense: copied
    w = c["w"].to(gpu).t().contiguous().t()
    _close(dense.linear(x, w, c["bias"].to(gpu), act="silu", residual=c["residual"].to(gpu)), ref, bound)
    y = dense.linear(c["x"].to(gpu).view(2, 3, 5, 64), c["w"].to(gpu), c["bias"].to(gpu), act="silu",
                     residual=c["residual"].to(gpu).view(2, 3, 5, 48))
    assert y.shape == (2, 3, 5, 48)
    _close(y.view(30, 48), ref, bound)
    y = dense.linear(c["x"].to(gpu)[4], c["w"].to(gpu), c["bias"].to(gpu), act="silu", residual=c["residual"].to(gpu)[4])
    assert y.shape == (48,)
    _close(y[None], ref[4:5], lambda d: bound(d)[4:5])
    assert dense.linear(c["x"].to(gpu)[:0], c["w"].to(gpu)).shape == (0, 48)


@pytest.mark.parametrize("M,K,N", [(5, 512, 96), (90, 6000, 64), (300, 128, 160)])
def test_residual_in_place(gpu, M, K, N):
    from ccut.quant import dense

    c = _inputs(M, K, N, BF, False, None, True, BF)
    r = c["residual"].to(gpu)
    assert dense.linear(c["x"].to(gpu), c["w"].to(gpu), residual=r, out=r) is r
    ref, bound = od.linear(c["x"], c["w"], residual=c["residual"])
    _close(r, ref, bound)
    with pytest.raises(ValueError, match="overlaps"):
        dense.linear(c["x"].to(gpu)[:-1], c["w"].to(gpu), residual=r[:-1], out=r[1:])


@pytest.mark.parametrize("M,K,N", [(4, 100, 40), (40, 256, 40), (100, 133, 40), (300, 192, 40)])
def test_not_finite(gpu, M, K, N):
    """Infinities and NaN stay in their own rows and columns, and give what the formula gives there."""
    from ccut.quant import dense

    c = _inputs(M, K, N, F16, False, None, False, F16)
    c["x"][1, 3] = float("inf")
    c["x"][M - 1, K - 1] = float("nan")
    c["w"][N - 1, 0] = float("-inf")
    for act in (None, "relu", "silu", "gelu", "gelu_tanh"):
        y = dense.linear(c["x"].to(gpu), c["w"].to(gpu), act=act).cpu().double()
        z = c["x"].double() @ c["w"].double().t()
        lin = torch.nn.functional
        ref = {None: z, "relu": torch.where(z < 0, 0.0, z), "silu": z / (1 + torch.exp(-z)),
               "gelu": 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5)), "gelu_tanh": lin.gelu(z, approximate="tanh")}[act]
        odd = ~torch.isfinite(z)
        assert torch.isfinite(y[~odd]).all()
        assert torch.equal(torch.isnan(y[odd]), torch.isnan(ref[odd]))
        inf = odd & torch.isinf(ref)
        assert torch.equal(y[inf], ref[inf])


def test_activations_far_out(gpu):
    """Every activation from the smallest to the largest pre-activations (K = 1: z is x)."""
    from ccut.quant import dense

    x = torch.cat([torch.linspace(-30, 30, 4001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 3e4, -3e4, 1e30, -1e30])])
    x = x.to(BF)[:, None]
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        for w in (1.0, 3e5):
            y = dense.linear(x.to(gpu), torch.full((1, 1), w, dtype=BF, device=gpu), act=act, out_dtype=F32)
            ref, bound = od.linear(x, torch.full((1, 1), w, dtype=BF), None, act)
            _close(y, ref, bound, act)


@pytest.mark.parametrize("T,k,E,K,N", [(1, 1, 1, 64, 48), (1, 8, 128, 256, 96), (16, 6, 64, 128, 160), (50, 4, 7, 130, 70),
                                       (64, 2, 4, 200, 33), (500, 8, 16, 256, 128), (300, 4, 4, 264, 264),
                                       (40, 2, 1024, 64, 32), (2000, 2, 8, 96, 256)])
@pytest.mark.parametrize("dt", [BF, F16])
def test_grouped(gpu, T, k, E, K, N, dt):
    from ccut.quant import dense

    g = torch.Generator().manual_seed(T + E)
    ids = torch.rand((T, E), generator=g).argsort(1)[:, :k].clone()
    ids[torch.rand((T, k), generator=g) < 0.1] = -1
    _, offsets = op.plan(ids, E)
    for gated, act, bias in ((False, None, "same"), (True, "silu", None), (True, "gelu", F32)):
        c = _inputs(T * k, K, N, dt, gated, bias, False, dt, E=E)
        ref, bound = od.grouped(c["x"], offsets, c["w"], c["bias"], act, gated)
        y = dense.linear_grouped(c["x"].to(gpu), offsets.to(gpu), c["w"].to(gpu), _up(c["bias"], gpu), act=act, gated=gated)
        _close(y, ref, bound)
        assert (y[int(offsets[-1]):] == 0).all()


@pytest.mark.parametrize("M,E,K,W", [(4536, 70, 136, 130), (1746, 16, 136, 912), (4134, 70, 280, 258), (4403, 40, 144, 1052),
                                     (4286, 40, 136, 1468)])
@pytest.mark.parametrize("gated,act,bias", [(False, "relu", "same"), (True, "silu", F32)])
def test_tiles_of_groups(gpu, M, E, K, W, gated, act, bias):
    """Sizes for each shape of tile, experts of uneven rows, K's last stage cut short, rows of no expert."""
    from ccut.quant import dense

    g = torch.Generator().manual_seed(M)
    cuts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.randint(0, M - 50, (E,), generator=g).sort().values])
    offsets = cuts.to(torch.int32)
    c = _inputs(M, K, W // 2 if gated else W, BF, gated, bias, False, BF, E=E)
    c["x"][int(offsets[-1]):] = float("nan")  # not read
    ref, bound = od.grouped(c["x"].nan_to_num(0.0), offsets, c["w"], c["bias"], act, gated)
    y = dense.linear_grouped(c["x"].to(gpu), offsets.to(gpu), c["w"].to(gpu), _up(c["bias"], gpu), act=act, gated=gated)
    _close(y, ref, bound)
    assert (y[int(offsets[-1]):] == 0).all()


@pytest.mark.parametrize("counts", [[0, 0, 0], [0, 5, 0], [200, 0, 1], [1, 1, 1], [16, 32, 64], [17, 33, 65], [0, 0, 700],
                                    [129, 256, 513], [300, 2, 0], [1500, 1, 0], [64] * 64])
def test_group_sizes(gpu, counts):
    """Groups of none, one and many rows, rows of no expert behind them, any alignment of rows and columns."""
    from ccut.quant import dense

    E, kept = len(counts), sum(counts)
    offsets = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
    for extra in (0, 1, 70, 333):
        for K, N in ((72, 40), (65, 33)):
            c = _inputs(kept + extra, K, N, BF, True, "same", False, F32, E=E)
            c["x"][kept:] = float("nan")  # not read
            wide = torch.full((kept + extra, N + 3), 7.0, dtype=F32, device=gpu)
            y = dense.linear_grouped(c["x"].to(gpu), offsets.to(gpu), c["w"].to(gpu), c["bias"].to(gpu), act="silu",
                                     gated=True, out=wide[:, 1:N + 1])
            ref, bound = od.grouped(c["x"], offsets, c["w"], c["bias"], "silu", True)
            _close(y, ref, bound)
            assert (y[kept:] == 0).all() and (wide[:, 0] == 7).all() and (wide[:, N + 1:] == 7).all()


@pytest.mark.parametrize("M,K,N", [(1300, 1031, 900), (700, 2049, 1500), (2100, 257, 1700), (513, 4100, 700)])
def test_large_unaligned(gpu, M, K, N):
    """Products large enough to copy their unaligned rows first: odd K, and K of whole pieces at odd addresses."""
    from ccut.quant import dense

    for gated, dt in ((False, BF), (True, F16)):
        c = _inputs(M, K, N // 2 if gated else N, dt, gated, "same", True, dt)
        _run(gpu, c, gated, "silu")
        K8 = K // 8 * 8
        c = _inputs(M, K8, N, dt, False, None, False, dt)
        ref, bound = od.linear(c["x"], c["w"])
        for dx, dw in ((1, 0), (0, 3), (5, 8)):
            x = torch.full((M * (K8 + 3) + 16,), float("nan"), dtype=dt, device=gpu)[dx:dx + M * (K8 + 3)].view(M, K8 + 3)[:, :K8]
            w = torch.empty((N * K8 + 16,), dtype=dt, device=gpu)[dw:dw + N * K8].view(N, K8)
            x.copy_(c["x"])
            w.copy_(c["w"])
            _close(dense.linear(x, w), ref, bound)


@pytest.mark.parametrize("E,rows,K,N", [(3, 900, 515, 700), (2, 700, 1030, 1100)])
def test_large_unaligned_groups(gpu, E, rows, K, N):
    from ccut.quant import dense

    counts = [rows, 0] + [rows // 3] * (E - 1)
    offsets = torch.tensor([0] + torch.tensor(counts[:E]).cumsum(0).tolist(), dtype=torch.int32)
    M = int(offsets[-1]) + 37
    c = _inputs(M, K, N, F16, True, F32, False, F16, E=E)
    c["x"][int(offsets[-1]):] = float("nan")
    ref, bound = od.grouped(c["x"], offsets, c["w"], c["bias"], "gelu", True)
    y = dense.linear_grouped(c["x"].to(gpu), offsets.to(gpu), c["w"].to(gpu), c["bias"].to(gpu), act="gelu", gated=True)
    _close(y, ref, bound)
    assert (y[int(offsets[-1]):] == 0).all()


def test_repeated_calls_give_the_same_bits(gpu):
    from ccut.quant import dense

    for M, K, N in ((3, 4096, 64), (100, 8192, 96), (300, 512, 256)):
        c = {k: _up(v, gpu) for k, v in _inputs(M, K, N, BF, False, None, True, BF).items()}
        first = dense.linear(c["x"], c["w"], act="gelu", residual=c["residual"])
        for _ in range(5):
            assert torch.equal(first, dense.linear(c["x"], c["w"], act="gelu", residual=c["residual"]))


def test_graphs_and_streams(gpu):
    """Captured calls with scratch of their own, two graphs, replayed with eager work between, against eager results."""
    from ccut.quant import dense

    shapes = [(100, 8192, 96), (90, 6000, 160), (4, 512, 64), (1300, 1031, 900)]
    cs = [{k: _up(v, gpu) for k, v in _inputs(M, K, N, BF, False, "same", False, BF).items()} for M, K, N in shapes]
    call = lambda c: dense.linear(c["x"], c["w"], c["bias"], act="silu")  # noqa: E731
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cs:
            call(c)
    torch.cuda.current_stream().wait_stream(side)
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    gen = torch.Generator().manual_seed(5)
    for _ in range(4):
        for c in cs:
            c["x"].copy_(torch.randn(c["x"].shape, generator=gen))
        want = [call(c) for c in cs]
        for g, o in zip(graphs, outs):
            o.fill_(float("nan"))
            g.replay()
        torch.cuda.synchronize()
        for o, y in zip(outs, want):
            assert torch.equal(o, y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [call(cs[0]) for _ in range(3)]
    torch.cuda.synchronize()
    for y in got:
        assert torch.equal(y, call(cs[0]))


@pytest.mark.parametrize("M,K,ldx", [(300, 128, (1 << 23) - 8), (300, 128, (1 << 23) + 8), (12, 128, (1 << 28) + 8),
                                     (40, 128, (1 << 23) + 8)])
def test_rows_far_apart(gpu, M, K, ldx):
    """Rows of x whose distance in a tile fits 32 bits by a little, and does not."""
    from ccut.quant import dense

    c = _inputs(M, K, 72, BF, False, None, False, BF)
    far = torch.empty((M - 1) * ldx + K, dtype=BF, device=gpu).as_strided((M, K), (ldx, 1))
    far.copy_(c["x"])
    ref, bound = od.linear(c["x"], c["w"], None, "silu")
    _close(dense.linear(far, c["w"].to(gpu), act="silu"), ref, bound)
    del far
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_weights_beyond_32_bits(gpu, rows):
    """The last of experts whose weights take 4.6 GiB, its rows and y behind 2^31 elements' worth of others."""
    from ccut.quant import dense

    E, K, N = 37, 4096, 8192
    c = _inputs(rows, K, N, BF, True, None, False, BF)
    w = torch.empty((E, 2 * N, K), dtype=BF, device=gpu)
    w[E - 1] = c["w"].to(gpu)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=gpu)
    offsets[E] = rows
    y = dense.linear_grouped(c["x"].to(gpu), offsets, w, act="silu", gated=True)
    ref, bound = od.linear(c["x"], c["w"], None, "silu", True)
    _close(y, ref, bound)
    del w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("M", [4, 40])
def test_gated_halves_beyond_32_bits(gpu, M):
    """The up half of w more than 2^31 elements behind the gate's."""
    from ccut.quant import dense

    K, N = 4096, (1 << 19) + 40
    g = torch.Generator().manual_seed(M)
    x, ws = torch.randn((M, K), generator=g).to(BF), (torch.randn((2, 24, K), generator=g) * K ** -0.5).to(BF)
    w = torch.zeros((2, N, K), dtype=BF, device=gpu)
    w[:, -24:] = ws.to(gpu)
    y = dense.linear(x.to(gpu), w.view(2 * N, K), act="silu", gated=True)
    ref, bound = od.linear(x, ws.reshape(48, K), None, "silu", True)
    _close(y[:, -24:], ref, bound)
    assert (y[:, :-24] == 0).all()
    del w, y
    torch.cuda.empty_cache()


def test_refusals(gpu):
    from ccut.quant import dense

    x, w = torch.zeros((4, 64), dtype=BF, device=gpu), torch.zeros((32, 64), dtype=BF, device=gpu)
    b, off = torch.zeros(32, device=gpu), torch.zeros(4, dtype=torch.int32, device=gpu)
    w3 = torch.zeros((3, 32, 64), dtype=BF, device=gpu)
    square = torch.zeros((64, 64), dtype=BF, device=gpu)
    for call in (lambda: dense.linear(x, square, out=square[8:12]),
                 lambda: dense.linear(x, square, torch.zeros(64, dtype=BF, device=gpu), out=square[:4]),
                 lambda: dense.linear(x[:1], w, b, out=b.view(1, 32), out_dtype=F32),
                 lambda: dense.linear_grouped(x[:1], off, w3, out=w3[2, 3:4, :32]),
                 lambda: dense.linear(x.float(), w), lambda: dense.linear(x, w.half()), lambda: dense.linear(x, w.cpu()),
                 lambda: dense.linear(x[:, :32], w), lambda: dense.linear(x, w[0]), lambda: dense.linear(x, w3),
                 lambda: dense.linear(x, w[:31], gated=True), lambda: dense.linear(x, w, act="tanh"),
                 lambda: dense.linear(x, w, b[:16]), lambda: dense.linear(x, w, b.double()),
                 lambda: dense.linear(x, w, b.cpu()), lambda: dense.linear(x, w, residual=x),
                 lambda: dense.linear(x, w, residual=torch.zeros((4, 32), device=gpu)),
                 lambda: dense.linear(x, w, out_dtype=torch.float64),
                 lambda: dense.linear(x, w, out=torch.zeros((4, 32), dtype=F16, device=gpu), out_dtype=BF),
                 lambda: dense.linear(x, w, out=torch.zeros((32, 4), dtype=BF, device=gpu).t()),
                 lambda: dense.linear(x, w, out=x[:, :32]), lambda: dense.linear(x.cpu(), w),
                 lambda: dense.linear(torch.zeros((1 << 20) + 1, 1, dtype=BF, device=gpu), w[:, :1]),
                 lambda: dense.linear_grouped(x, None, w3), lambda: dense.linear_grouped(x, off.long(), w3),
                 lambda: dense.linear_grouped(x, off[:3], w3), lambda: dense.linear_grouped(x, off.cpu(), w3),
                 lambda: dense.linear_grouped(x, off, w), lambda: dense.linear_grouped(x[None], off, w3),
                 lambda: dense.linear_grouped(x, off, w3, b), lambda: dense.linear_grouped(x, off[:1], w3[:0])):
        with pytest.raises(ValueError):
            call()
