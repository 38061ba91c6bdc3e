"""``quant.dense.linear`` and ``linear_grouped`` on each of their kernels, tiles,
splits of K and aligned copies: sizes for each, the rule's choice (host code: no
GPU is needed), and the products on the GPU.

The products are of small whole numbers, so every sum in float32 is exact in any
order and the results have to be equal: one term lost or taken twice shows,
however long K is.  With |x|, |w| <= 2 sums stay within 4 K < 2^24."""

from __future__ import annotations

import ctypes

import pytest
import torch

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FEW, MID, RING, TILE, RAGGED = range(5)
X, W, BOTH = 1, 2, 3  # what is copied to aligned rows


def _route(lib, M, K, rows, gated=False, E=0, dx=0, dw=0, pad=0):
    """(kernel, rows and columns of a workgroup, splits, copies) of ``rows`` rows of w, x and w ``dx`` and ``dw``
    elements behind a 256-byte boundary, x's rows ``pad`` elements apart."""
    from ccut._lib import DENSE_ARGS

    N = rows // 2 if gated else rows
    got = [ctypes.c_int() for _ in range(4)]
    args = DENSE_ARGS.pack(256 + 2 * dx, 256 + 2 * dw, 0, 0, 256, 256, 0, 0, 0, K + pad, N, N, M, K, N, E, 2, 0, 2, 0, gated)
    kernel = lib.ccq_dense_linear_kernel(args, E > 0, *map(ctypes.byref, got))
    return kernel, *(v.value for v in got)


def _whole(g, shape, largest=2):
    return torch.randint(-largest, largest + 1, shape, generator=g, dtype=torch.int8)


def _amid_nan(t, gpu, dt, shift=0, pad=0):
    """``t [rows, width]`` on the GPU, ``shift`` elements into a buffer of NaN, its rows ``pad`` elements apart."""
    rows, width = t.shape
    buf = torch.full((rows * (width + pad) + shift + 64,), float("nan"), dtype=dt, device=gpu)
    return buf[shift:shift + rows * (width + pad)].view(rows, width + pad)[:, :width].copy_(t)


def _finish(z, bias, N, gated, act, residual):
    z = z.double()
    if bias is not None:
        z = z + bias
    g = z[:, :N].clamp_min(0) if act == "relu" else z[:, :N]
    if gated:
        g = g * z[:, N:]
    if residual is not None:
        g = g + residual
    assert g.abs().max() < 2 ** 24  # exact in float32
    return g


def _check(gpu, M, K, rows, gated, dt, ydt, act=None, bias=False, residual=False, E=0, dx=0, dw=0, pad=0):
    from ccut.quant import dense

    g = torch.Generator().manual_seed(M * 31 + K * 7 + rows + gated)
    N = rows // 2 if gated else rows
    rows = 2 * N if gated else N
    L = max(E, 1)
    x, w = _whole(g, (M, K)).float(), _whole(g, (L, rows, K)).float()
    b = _whole(g, (L, rows), 5) if bias else None
    r = _whole(g, (M, N), 9) if residual else None
    xd = _amid_nan(x, gpu, dt, dx, pad)
    wd = _amid_nan(w.view(L * rows, K), gpu, dt, dw).view(L, rows, K)
    bd = b.float().to(gpu) if bias else None
    want = torch.zeros((M, N), dtype=torch.float64)
    if E:
        # uneven groups, empty ones, rows of no expert behind them (NaN: they do not count)
        cuts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.randint(0, M - 50, (E,), generator=g).sort().values])
        cuts[E // 2] = cuts[E // 2 + 1]
        for e in range(E):
            n, m = int(cuts[e]), int(cuts[e + 1])
            if n < m:
                want[n:m] = _finish(x[n:m] @ w[e].t(), b[e] if bias else None, N, gated, act, None)
        xd[int(cuts[E]):] = float("nan")
        y = dense.linear_grouped(xd, cuts.to(torch.int32).to(gpu), wd, bd, act=act, gated=gated, out_dtype=ydt)
    else:
        want = _finish(x @ w[0].t(), b[0] if bias else None, N, gated, act, r)
        y = dense.linear(xd, wd[0], bd[0] if bias else None, act=act, gated=gated,
                         residual=r.to(ydt).to(gpu) if residual else None, out_dtype=ydt)
    want = want.float().to(ydt)
    same = y.cpu() == want
    assert same.all(), f"{(~same).sum()} of {same.numel()} differ, the first at {(~same).nonzero()[0].tolist()}"


# ---- rows at any alignment: products large enough to copy x, w or both to aligned rows first
COPIED = [
    (2100, 257, 1700, 0, {}, (RING, 128, 128, 1, BOTH)), (2000, 520, 1900, 0, dict(dx=1), (RING, 128, 128, 1, X)),
    (2000, 520, 1900, 0, dict(dw=3), (RING, 128, 128, 1, W)), (2000, 520, 1900, 0, dict(pad=3), (RING, 128, 128, 1, X)),
    (1500, 1032, 2000, 0, dict(dx=5, dw=2), (RING, 128, 128, 1, BOTH)), (2600, 1416, 2200, 0, dict(dw=1), (RING, 256, 128, 1, W)),
    (700, 2049, 1500, 0, dict(dx=1, dw=1), (RING, 64, 64, 1, BOTH)),
    (4000, 515, 700, 2, {}, (RING, 128, 128, 1, BOTH)), (4000, 520, 700, 2, dict(dx=3), (RING, 128, 128, 1, X)),
    (4000, 520, 700, 2, dict(dw=1), (RING, 128, 128, 1, W)), (2500, 1030, 900, 3, dict(pad=5), (RING, 128, 128, 1, BOTH)),
    (6628, 657, 1736, 5, dict(dx=1, dw=1), (TILE, 256, 256, 1, BOTH)),
]


# as measured: unaligned tiles take 38 and 59 us for the first two, copies and aligned ones 31 and 48; unaligned ones
# 17.9 and 13.5 us for the others, copies 20.9 and 21
UNALIGNED = [(1274, 2747, 1520, (RING, 64, 64, 1, BOTH)), (346, 5468, 4379, (RING, 128, 128, 2, BOTH)),
             (293, 2355, 1447, (RAGGED, 64, 64, 4, 0)), (54, 6003, 1305, (RAGGED, 64, 64, 12, 0))]


@pytest.fixture(scope="module")
def lib(built_lib):
    from ccut import _lib

    return _lib.lib()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,rows,E,at,route", COPIED)
def test_choice_copied(lib, M, K, rows, E, at, route, gated):
    assert _route(lib, M, K, rows, gated, E, **at) == route


@pytest.mark.parametrize("M,K,N,route", UNALIGNED)
def test_choice_unaligned(lib, M, K, N, route):
    assert _route(lib, M, K, N) == route


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N,route", UNALIGNED)
def test_unaligned(gpu, M, K, N, route):
    _check(gpu, M, K, N, False, BF, BF, bias=True, residual=True)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,rows,E,at,route", COPIED)
def test_copied(gpu, M, K, rows, E, at, route, gated):
    _check(gpu, M, K, rows, gated, F16 if gated else BF, F32 if gated else BF, "relu" if gated else None, bias=True,
           residual=not E, E=E, **at)


@pytest.mark.gpu
def test_copies_in_graphs(gpu):
    """Two captured calls whose scratch holds the aligned copies, a batch's and experts': replays with eager calls
    between them against these."""
    from ccut.quant import dense

    g = torch.Generator().manual_seed(2)
    offsets = torch.tensor([0, 2900, 3950], dtype=torch.int32, device=gpu)
    state = []
    for M, K, rows, E in ((2100, 257, 1700, 0), (4000, 515, 700, 2)):
        x = _whole(g, (M, K)).to(BF).to(gpu)
        w = _whole(g, (E, rows, K) if E else (rows, K)).to(BF).to(gpu)
        call = (lambda x=x, w=w: dense.linear_grouped(x, offsets, w)) if E else (lambda x=x, w=w: dense.linear(x, w))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call()
        state.append((graph, y, call, x))
    for _ in range(4):
        want = []
        for _, y, call, x in state:
            x.copy_(_whole(g, x.shape))
            want.append(call())
            y.fill_(float("nan"))
        for graph, *_ in state:
            graph.replay()
        torch.cuda.synchronize()
        for (_, y, _, _), ref in zip(state, want):
            assert torch.equal(y, ref)


# ---- tiles whose ring of stages goes round several times: K of ten stages or more, the last one whole or cut short,
# and (groups) experts of uneven rows, so that waves behind a short tile's end only copy.  The second route is the
# gated product's, where another one is taken.
WIDE = (TILE, 256, 224, 1, 0), (TILE, 256, 256, 1, 0)
TILED = [
    (513, 640, 12416, 0, [(TILE, 128, 128, 1, 0)]), (513, 712, 12410, 0, [(TILE, 128, 128, 1, 0)]),
    (530, 648, 14300, 0, [(TILE, 256, 192, 1, 0)]), (900, 2048, 9000, 0, [(TILE, 256, 192, 1, 0)]),
    (900, 648, 12416, 0, WIDE), (777, 712, 14200, 0, WIDE), (2050, 640, 6272, 0, WIDE), (40, 712, 9000, 0, [(RING, 64, 64, 1, 0)]),
    (1000, 648, 2050, 0, [(RING, 128, 128, 1, 0)]), (600, 1288, 9000, 0, [(RING, 256, 128, 1, 0)]),
    (60, 1288, 8100, 0, [(MID, 32, 64, 1, 0)]),
    (300, 712, 450, 128, [(TILE, 128, 128, 1, 0)]), (3000, 712, 1468, 12, [(TILE, 128, 128, 1, 0)]),
    (4403, 712, 1052, 40, [(TILE, 256, 192, 1, 0)]), (4403, 640, 1052, 40, [(TILE, 256, 192, 1, 0)]),
    (4286, 712, 1468, 40, [(TILE, 256, 256, 1, 0)]), (2500, 648, 1468, 40, [(TILE, 256, 256, 1, 0)]),
    (4134, 712, 258, 70, [(RING, 128, 128, 1, 0)]), (2500, 1288, 1468, 8, [(RING, 128, 128, 1, 0)]),
    (1746, 712, 130, 70, [(RING, 64, 64, 1, 0)]), (1000, 648, 130, 70, [(MID, 32, 64, 1, 0)]),
]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,rows,E,routes", TILED)
def test_choice_tiled(lib, M, K, rows, E, routes, gated):
    assert _route(lib, M, K, rows, gated, E) == routes[-1 if gated else 0]


@pytest.mark.gpu
@pytest.mark.parametrize("ydt", [BF, F32])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,rows,E,routes", TILED)
def test_tiled(gpu, M, K, rows, E, routes, gated, ydt):
    _check(gpu, M, K, rows, gated, BF, ydt, "relu" if gated else None, bias=True, residual=not E, E=E)


# ---- K shared by several workgroups, its parts whole and cut short
SPLIT = [
    (64, 4096, 4096, {}, (RING, 64, 64, 4, 0)), (64, 4104, 4100, {}, (RING, 64, 64, 6, 0)),
    (40, 14336, 4096, {}, (RING, 64, 64, 8, 0)), (128, 4104, 4100, {}, (RING, 128, 128, 5, 0)),
    (172, 4096, 4096, {}, (RING, 128, 128, 4, 0)), (300, 7176, 2050, {}, (RING, 128, 128, 5, 0)),
    (400, 14336, 1024, {}, (RING, 128, 128, 8, 0)), (172, 7176, 9000, {}, (RING, 256, 128, 3, 0)),
    (90, 14336, 12416, {}, (TILE, 128, 128, 5, 0)), (20, 14336, 256, {}, (MID, 32, 64, 16, 0)),
    (50, 14329, 520, dict(dx=1), (RAGGED, 64, 64, 16, 0)), (172, 10001, 1024, dict(dw=1, pad=2), (RAGGED, 64, 64, 10, 0)),
]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,rows,at,route", SPLIT)
def test_choice_split(lib, M, K, rows, at, route, gated):
    assert _route(lib, M, K, rows, gated, **at) == route


@pytest.mark.gpu
@pytest.mark.parametrize("ydt", [BF, F32])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K,rows,at,route", SPLIT)
def test_split(gpu, M, K, rows, at, route, gated, ydt):
    _check(gpu, M, K, rows, gated, F16, ydt, "relu" if gated else None, bias=True, residual=True, **at)


# ---- up to 16 rows: 16, 32 and 64 columns a workgroup, rows in whole eights, at dwords and at odd elements, K of less
# than one step of the waves, of whole steps and cut short (a step is 256 columns, of 64 columns a workgroup 128; four
# and two waves take steps in turn)
COLUMNS = [(70, 0, 16), (5200, 0, 32), (10300, 0, 64), (72, 3, 16), (2000, 3, 32), (4100, 3, 64)]


@pytest.mark.parametrize("rows,E,columns", COLUMNS)
def test_choice_few(lib, rows, E, columns):
    for K in (257, 1030, 4999, 2056):
        if E and K % 8 == 0 and rows > 2000:  # (aligned groups of that many tiles take others)
            continue
        assert _route(lib, 13, K, rows, False, E) == (FEW, 16, columns, 1, 0)
        assert _route(lib, 13, K, rows, True, E) == (FEW, 16, max(columns, 32), 1, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [257, 1024, 1030, 2049, 2056, 4999])
@pytest.mark.parametrize("rows,E,columns", COLUMNS)
def test_few(gpu, rows, E, columns, K):
    for i, (dx, dw, pad) in enumerate(((0, 0, 0), (1, 0, 0), (0, 1, 2), (3, 1, 1), (2, 2, 2))):
        for gated in (False, True):
            if E:
                _check_few_groups(gpu, K, rows, gated, E, dx, dw, pad)
            else:
                _check(gpu, (1, 5, 16)[i % 3], K, rows, gated, BF, (BF, F32)[i % 2], "relu" if gated else None,
                       bias=True, residual=i != 1, dx=dx, dw=dw, pad=pad)


def _check_few_groups(gpu, K, rows, gated, E, dx, dw, pad):
    """13 rows: nine and two of the outer experts', two of none."""
    from ccut.quant import dense

    g = torch.Generator().manual_seed(K + rows + gated)
    N = rows // 2 if gated else rows
    x, w, b = _whole(g, (13, K)).float(), _whole(g, (E, rows, K)).float(), _whole(g, (E, rows), 5)
    offsets = torch.tensor([0, 9] + [9] * (E - 2) + [11], dtype=torch.int32)
    want = torch.zeros((13, N), dtype=torch.float64)
    for e, n, m in ((0, 0, 9), (E - 1, 9, 11)):
        want[n:m] = _finish(x[n:m] @ w[e].t(), b[e], N, gated, "relu", None)
    xd, wd = _amid_nan(x, gpu, F16, dx, pad), _amid_nan(w.view(E * rows, K), gpu, F16, dw).view(E, rows, K)
    xd[11:] = float("nan")
    y = dense.linear_grouped(xd, offsets.to(gpu), wd, b.float().to(gpu), act="relu", gated=gated, out_dtype=F32)
    assert torch.equal(y.cpu(), want.float())
