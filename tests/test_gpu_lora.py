"""Adapters of many requests beside one projection (``ccq_lora_add``) against
the 64-bit product, element by element within the bound that the rounding of
float32 sums, of p's parts and of y allows (``oracle.lora``)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import lora as ol

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _case(T, K, N, R, L, xdt, wdt, ydt, seed=0, pattern="mixed", ranks=False, scale=True):
    g = torch.Generator().manual_seed(seed * 7919 + T * 131 + K * 17 + N * 3 + R)
    c = dict(x=torch.randn((T, K), generator=g).to(DT[xdt]), y=torch.randn((T, N), generator=g).to(DT[ydt]),
             a=(torch.randn((L, R, K), generator=g) * K ** -0.5).to(DT[wdt]),
             b=(torch.randn((L, N, R), generator=g) * 0.3).to(DT[wdt]), scale=None, rank=None)
    if scale:
        c["scale"] = torch.randn(L, generator=g)
    if ranks:
        c["rank"] = torch.randint(0, R + 1, (L,), generator=g, dtype=torch.int32)
    if pattern == "mixed":      # any adapter or none
        c["index"] = torch.randint(-1, L, (T,), generator=g)
    elif pattern == "runs":     # prompts one behind the other
        c["index"] = torch.sort(torch.randint(-1, L, (T,), generator=g)).values
    elif pattern == "one":
        c["index"] = torch.full((T,), L - 1)
    elif pattern == "none":
        c["index"] = torch.full((T,), -1)
    else:                       # beyond the adapters on both sides
        c["index"] = torch.randint(-3, L + 3, (T,), generator=g)
        c["index"][::5] = 2 ** 40
    return c


def _adapters(c, gpu):
    from ccut.quant import lora

    up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    return lora.LoraAdapters(up(c["a"]), up(c["b"]), up(c["scale"]), up(c["rank"]))


def _check(y, c):
    ref, bound = ol.add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"], c["rank"])
    off = (y.cpu().double() - ref).abs()
    tol = bound(c["y"].dtype, c["a"].dtype)
    assert torch.isfinite(y).all()
    assert (off <= tol).all(), f"worst {(off / tol).max():.3f} of the bound"
    bare = (c["index"] < 0) | (c["index"] >= c["a"].shape[0])
    assert torch.equal(y.cpu()[bare], c["y"][bare])


def _run(c, gpu):
    from ccut.quant import lora

    y = c["y"].to(gpu)
    got = lora.add_(y, c["x"].to(gpu), _adapters(c, gpu), c["index"].to(gpu))
    assert got is y
    return y


TYPES = [("bf16", "bf16", "bf16"), ("f16", "f16", "f16"), ("f32", "bf16", "f32"), ("f32", "f16", "f32"),
         ("bf16", "bf16", "f32"), ("f16", "f16", "f32"), ("bf16", "f16", "bf16"), ("f16", "bf16", "f16"),
         ("f32", "bf16", "bf16")]


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("T,K,N,R,L", [(1, 256, 320, 16, 3), (16, 512, 1024, 8, 4), (17, 160, 65, 32, 2),
                                       (70, 1405, 257, 12, 9), (300, 384, 192, 64, 5)])
def test_types(gpu, T, K, N, R, L, types):
    c = _case(T, K, N, R, L, *types)
    _check(_run(c, gpu), c)


@pytest.mark.parametrize("R", [1, 2, 5, 8, 15, 16, 17, 24, 31, 32, 33, 48, 64, 65, 100, 128, 129, 200, 256])
def test_ranks(gpu, R):
    for T, t in ((3, "bf16"), (33, "f16")):
        c = _case(T, 200, 136, R, 3, t, t, t)
        _check(_run(c, gpu), c)


@pytest.mark.parametrize("K", [1, 3, 7, 8, 9, 31, 32, 33, 127, 128, 129, 513, 4096, 14336])
def test_inner_sizes(gpu, K):
    for T, t in ((1, "bf16"), (20, "f16"), (5, "f32")):
        c = _case(T, K, 80, 16, 2, t, "bf16" if t == "f32" else t, t)
        _check(_run(c, gpu), c)


def test_smallest_buffers(gpu):
    """Fewer values than one load takes, and barely as many."""
    for T, K, N, R, L in ((1, 1, 1, 1, 1), (1, 7, 40, 3, 2), (1, 8, 40, 3, 2), (2, 3, 9, 5, 1), (3, 300, 1, 1, 7),
                          (3, 300, 1, 1, 8), (5, 1, 77, 7, 1), (5, 2, 77, 4, 1), (2000, 1, 3, 1, 2), (700, 5, 2, 3, 2)):
        for t in ("bf16", "f16", "f32"):
            c = _case(T, K, N, R, L, t, "bf16" if t == "f32" else t, t)
            _check(_run(c, gpu), c)


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000, 14336])
def test_outer_sizes(gpu, N):
    for T, t in ((1, "bf16"), (20, "f16"), (5, "f32")):
        c = _case(T, 96, N, 16, 2, t, "f16" if t == "f32" else t, t)
        _check(_run(c, gpu), c)


@pytest.mark.parametrize("pattern", ["mixed", "runs", "one", "none", "beyond"])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 128, 255, 256, 257, 1000, 2049, 4097])
def test_batches(gpu, T, pattern):
    for L in (1, 7, 130):
        c = _case(T, 64, 72, 8, L, "bf16", "bf16", "bf16", pattern=pattern)
        _check(_run(c, gpu), c)


def test_most_adapters_and_tokens(gpu):
    c = _case(2000, 64, 48, 4, 1024, "f16", "f16", "f16")
    _check(_run(c, gpu), c)
    c = _case(65536, 32, 24, 4, 40, "bf16", "bf16", "bf16", pattern="runs")
    _check(_run(c, gpu), c)


@pytest.mark.parametrize("T", [40, 600, 1111])
@pytest.mark.parametrize("types", TYPES, ids="-".join)
def test_high_ranks_and_long_rows(gpu, T, types):
    """Ranks and rows that go through two kernels at any number of tokens."""
    for K, N, R in ((2056, 200, 256), (4100, 96, 130), (9000, 72, 40)):
        c = _case(T, K, N, R, 3, *types, pattern="runs" if T > 600 else "mixed", ranks=T == 600)
        _check(_run(c, gpu), c)


def test_padded_ranks_are_not_read(gpu):
    """Ranks 0 to R; what is behind an adapter's rank is NaN."""
    for R, t in ((16, "bf16"), (40, "f16"), (128, "bf16")):
        c = _case(90, 136, 100, R, 12, t, t, t, ranks=True)
        c["rank"][0], c["rank"][1], c["rank"][2] = 0, R, 1
        c["rank"][3] = R + 5     # clamped
        ref = {k: v.clone() if v is not None else None for k, v in c.items()}
        for i, r in enumerate(c["rank"].tolist()):
            c["a"][i, r:] = float("nan")
            c["b"][i, :, r:] = float("inf")
        _check(_run(c, gpu), ref)


def test_not_finite_stays_in_its_row(gpu):
    for t in ("bf16", "f16", "f32"):
        c = _case(40, 96, 70, 16, 3, t, "bf16" if t == "f32" else t, t, pattern="one")
        c["index"][7] = -1
        clean = _run(c, gpu)
        c["x"][3, 5] = float("nan")
        c["x"][9] = float("inf")
        c["x"][7] = float("nan")  # has no adapter
        y = _run(c, gpu)
        rows = torch.ones(40, dtype=torch.bool)
        rows[[3, 9]] = False
        assert torch.equal(y.cpu()[rows], clean.cpu()[rows])
        assert y[3].isnan().all() and not torch.isfinite(y[9]).any()


def test_half_range(gpu):
    """Inner products far beyond float16's range, and far below it."""
    for factor in (2.0 ** 9, 2.0 ** -9):
        c = _case(37, 2048, 64, 16, 2, "f16", "f16", "f32", scale=False)
        c["x"] = c["x"] * factor
        c["a"] = c["a"] * factor
        c["b"] = (c["b"].float() / factor).half()
        _check(_run(c, gpu), c)


def test_views_of_larger_buffers(gpu):
    """x and y as columns of one buffer at odd offsets, guarded on all sides;
    leading dimensions; an int32 index."""
    from ccut.quant import lora

    for K, N, off in ((100, 77, 1), (256, 192, 3), (64, 128, 8)):
        c = _case(24, K, N, 16, 4, "bf16", "bf16", "bf16")
        big = torch.full((26, K + N + 20), 5.0, dtype=torch.bfloat16, device=gpu)
        xs, ys = big[1:25, off:off + K], big[1:25, off + K:off + K + N]
        xs.copy_(c["x"].to(gpu))
        ys.copy_(c["y"].to(gpu))
        before = big.clone()
        lora.add_(ys, xs, _adapters(c, gpu), c["index"].to(gpu).to(torch.int32))
        _check(ys, c)
        ys.copy_(c["y"].to(gpu))
        assert torch.equal(big, before)
    c = _case(24, 64, 48, 8, 4, "f16", "f16", "f16")
    y = c["y"].to(gpu).view(2, 3, 4, 48)
    lora.add_(y, c["x"].to(gpu).view(2, 3, 4, 64), _adapters(c, gpu), c["index"].to(gpu).view(2, 3, 4))
    _check(y.view(24, 48), c)
    none = torch.empty((0, 48), dtype=torch.float16, device=gpu)
    assert lora.add_(none, torch.empty((0, 64), dtype=torch.float16, device=gpu), _adapters(c, gpu),
                     torch.empty(0, dtype=torch.int64, device=gpu)) is none
    turned = c["x"].to(gpu).t().contiguous().t()  # rows that are columns
    y = c["y"].to(gpu)
    lora.add_(y, turned, _adapters(c, gpu), c["index"].to(gpu))
    _check(y, c)


def test_replaced_in_place(gpu):
    """An adapter replaced in the stack is used by the next call."""
    from ccut.quant import lora

    c = _case(30, 128, 96, 16, 3, "bf16", "bf16", "bf16")
    ad = _adapters(c, gpu)
    lora.add_(c["y"].to(gpu), c["x"].to(gpu), ad, c["index"].to(gpu))
    c["a"][1], c["b"][1] = c["a"][1].flip(1), c["b"][1].flip(0)
    ad.a[1].copy_(c["a"][1])
    ad.b[1].copy_(c["b"][1])
    _check(lora.add_(c["y"].to(gpu), c["x"].to(gpu), ad, c["index"].to(gpu)), c)


@pytest.mark.parametrize("T", [5, 90, 700])
def test_captured_and_two_streams(gpu, T):
    """A captured call replays on new inputs like the eager one, with eager
    work between the replays; two graphs and two streams at once; the same
    bits every time."""
    from ccut.quant import lora

    cs = [_case(T, 320, 200, 16, 6, "bf16", "bf16", "bf16", seed=s, ranks=True) for s in range(4)]
    ads = [_adapters(c, gpu) for c in cs]
    eager = [_run(c, gpu) for c in cs]
    for c, y in zip(cs, eager):
        _check(y, c)
    graphs = []
    for n in range(2):  # each on its own adapters
        x, y, index = cs[n]["x"].to(gpu), cs[n]["y"].to(gpu), cs[n]["index"].to(gpu)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lora.add_(y, x, ads[n], index)
        graphs.append((graph, x, y, index))
    for turn in range(4):
        for n, (graph, x, y, index) in enumerate(graphs):
            src = cs[(n + 2 * turn) % 4]
            x.copy_(src["x"].to(gpu))
            y.copy_(src["y"].to(gpu))
            index.copy_(src["index"].to(gpu))
        torch.cuda.synchronize()
        graphs[0][0].replay()
        graphs[1][0].replay()
        for n, (graph, x, y, index) in enumerate(graphs):
            src = cs[(n + 2 * turn) % 4]
            want = lora.add_(src["y"].to(gpu), src["x"].to(gpu), ads[n], src["index"].to(gpu))
            torch.cuda.synchronize()
            assert torch.equal(y, want), f"turn {turn}, graph {n}"
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(5):
        ys = [c["y"].to(gpu) for c in cs[:2]]
        xs = [c["x"].to(gpu) for c in cs[:2]]
        ids = [c["index"].to(gpu) for c in cs[:2]]
        for n, st in enumerate(streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                lora.add_(ys[n], xs[n], ads[n], ids[n])
        torch.cuda.synchronize()
        assert all(torch.equal(ys[n], eager[n]) for n in range(2)), f"turn {turn}"


def test_far_adapters_and_rows(gpu):
    """Offsets beyond 2^31 elements in the stacks and in y."""
    from ccut.quant import lora

    L, R, K, N = 520, 256, 16640, 64
    a = torch.empty((L, R, K), dtype=torch.bfloat16, device=gpu)  # only the adapters in use are set
    b = torch.empty((L, N, R), dtype=torch.bfloat16, device=gpu)
    assert a.numel() > 2 ** 31
    g = torch.Generator(device=gpu).manual_seed(3)
    for i in (0, L - 1):
        a[i] = torch.randn((R, K), generator=g, device=gpu) * K ** -0.5
        b[i] = torch.randn((N, R), generator=g, device=gpu)
    x = torch.randn((6, K), generator=g, device=gpu).bfloat16()
    y = torch.randn((6, N), generator=g, device=gpu).bfloat16()
    index = torch.tensor([0, L - 1, -1, L - 1, 0, L], device=gpu)
    pick = lambda t: torch.stack([t[0], t[L - 1]]).cpu()  # noqa: E731
    c = dict(x=x.cpu(), y=y.cpu(), a=pick(a), b=pick(b), scale=None, rank=None,
             index=torch.tensor([0, 1, -1, 1, 0, 2]))
    lora.add_(y, x, lora.LoraAdapters(a, b), index)
    _check(y, c)
    del a, b
    T, ld = 36000, 65536
    buf = torch.empty((T, ld), dtype=torch.bfloat16, device=gpu)
    ys = buf[:, 11:11 + 40]
    c = _case(T, 32, 40, 8, 3, "bf16", "bf16", "bf16")
    ys.copy_(c["y"].to(gpu))
    lora.add_(ys, c["x"].to(gpu), _adapters(c, gpu), c["index"].to(gpu))
    _check(ys, c)


def test_refusals(gpu):
    from ccut.quant import lora

    def z(*s, dtype=torch.bfloat16):
        return torch.zeros(s, dtype=dtype, device=gpu)

    ad = lora.LoraAdapters(z(3, 8, 64), z(3, 48, 8))
    i = torch.zeros(5, dtype=torch.int64, device=gpu)
    both = z(5, 96)
    bad = [
        lambda: lora.LoraAdapters(z(3, 8, 64), z(3, 48, 9)),
        lambda: lora.LoraAdapters(z(3, 8, 64), z(2, 48, 8)),
        lambda: lora.LoraAdapters(z(8, 64), z(48, 8)),
        lambda: lora.LoraAdapters(z(3, 8, 64), z(3, 48, 8, dtype=torch.float16)),
        lambda: lora.LoraAdapters(z(3, 8, 64, dtype=torch.float32), z(3, 48, 8, dtype=torch.float32)),
        lambda: lora.LoraAdapters(z(1, 257, 64), z(1, 48, 257)),
        lambda: lora.LoraAdapters(z(1025, 1, 8), z(1025, 8, 1)),
        lambda: lora.LoraAdapters(z(0, 8, 64), z(0, 48, 8)),
        lambda: lora.LoraAdapters(z(3, 8, 64).cpu(), z(3, 48, 8)),
        lambda: lora.LoraAdapters(z(3, 8, 64), z(3, 48, 8).cpu()),
        lambda: lora.LoraAdapters(z(3, 8, 64), z(3, 48, 8), scale=torch.ones(2)),
        lambda: lora.LoraAdapters(z(3, 8, 64), z(3, 48, 8), rank=[8]),
        lambda: lora.add_(z(5, 47), z(5, 64), ad, i),
        lambda: lora.add_(z(5, 48), z(5, 63), ad, i),
        lambda: lora.add_(z(5, 48), z(4, 64), ad, i),
        lambda: lora.add_(z(5, 48), z(5, 64), ad, i[:4]),
        lambda: lora.add_(z(5, 48), z(5, 64), ad, i.float()),
        lambda: lora.add_(z(5, 48), z(5, 64), ad, i.cpu()),
        lambda: lora.add_(z(5, 48).cpu(), z(5, 64), ad, i),
        lambda: lora.add_(z(5, 48), z(5, 64).cpu(), ad, i),
        lambda: lora.add_(z(5, 48, dtype=torch.float64), z(5, 64), ad, i),
        lambda: lora.add_(z(5, 48), z(5, 64, dtype=torch.float64), ad, i),
        lambda: lora.add_(z(48, 5).t(), z(5, 64), ad, i),
        lambda: lora.add_(z(1, 48).expand(5, 48), z(5, 64), ad, i),
        lambda: lora.add_(z(65537, 48), z(65537, 64), ad, torch.zeros(65537, dtype=torch.int64, device=gpu)),
        lambda: lora.add_(both[:, :48], both[:, 32:], ad, i),
        lambda: lora.add_(both[:, 30:78], both[:, :64], ad, i),
    ]
    for n, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print(f"call {n} was not refused")


def test_beside_quantized_projections(gpu):
    """Norm, shared 8-bit projection and adapters, as a layer runs them: the
    FP8 chain against the same chain on act_quant's rows, the INT8 chain
    against its 64-bit product, LinearProj with adapters against apply and the
    adapters' product."""
    from ccut import workloads
    from ccut.blocks import norm
    from ccut.quant import fp8_block, int8, lora
    from ccut.quant.linear import FakeWeightReader, LinearProj

    T, H, N, R, L = 75, 512, 384, 16, 5
    g = torch.Generator(device=gpu).manual_seed(0)
    x, res = (torch.randn((T, H), generator=g, device=gpu).bfloat16() for _ in range(2))
    w = (1 + 0.1 * torch.randn(H, generator=g, device=gpu)).bfloat16()
    wq, ws = workloads.fp8_block_weights(1, N, H, 1, gpu)
    lin = fp8_block.prepare(wq[0], ws[0], H)
    c = _case(T, H, N, R, L, "bf16", "bf16", "bf16")
    ad, index = _adapters(c, gpu), c["index"].to(gpu)

    q, scale, y, res2 = norm.rms_norm_fp8(x, w, residual=res, normed=True)
    out = fp8_block.linear_quantized(lin, q, scale, torch.bfloat16)
    base = out.clone()
    lora.add_(out, y, ad, index)
    # the codes and scales stand for the normalized rows to half a step of e4m3
    deq = (q.view(torch.float8_e4m3fn).double().view(T, -1, 128) * scale.double()[..., None]).view(T, H)
    exact = on_norm(x, w, res)
    amax = exact.abs().view(T, -1, 128).amax(-1, keepdim=True).expand(T, H // 128, 128).reshape(T, H)
    assert ((deq - exact).abs() <= exact.abs() * (2.0 ** -4 + 1e-5) + amax / 448 * 2.0 ** -10 * 1.01).all()
    # the same GEMM on the same codes: bit by bit what the linear on act_quant's rows gives for them
    aq, asc = fp8_block.act_quant(y)
    assert torch.equal(fp8_block.linear_quantized(lin, aq, asc), fp8_block.linear(lin, None, y))
    cc = dict(c, x=y.cpu(), y=base.cpu())
    _check(out, cc)

    i8 = norm.rms_norm_int8(x, w, residual=res, normed=True)
    wi = torch.randint(-127, 128, (N, H), generator=g, device=gpu, dtype=torch.int8)
    wsc = torch.rand(N, generator=g, device=gpu) * 0.01
    out = int8.int8_linear(i8.q, i8.scale, wi, wsc)
    ref = (i8.q.double() @ wi.double().t()) * i8.scale.double()[:, None] * wsc.double()
    assert ((out.double() - ref).abs() <= 3 * 2.0 ** -24 * ref.abs()).all()
    base = out.clone()
    lora.add_(out, i8.y, ad, index)
    _check(out, dict(c, x=i8.y.cpu(), y=base.cpu()))

    rng = np.random.default_rng(0)
    wf = rng.standard_normal((N, H)).astype(np.float32) * 0.05
    reader = FakeWeightReader({(0, "proj"): wf.tobytes()}, {(0, "proj"): (N, H, "F32")})
    proj = LinearProj(0, "proj", N, H, reader, None)
    xf = rng.standard_normal((T, H)).astype(np.float32)
    plain = proj.apply(xf)
    got = proj.apply(xf, adapters=ad, index=c["index"].numpy())
    assert isinstance(got, np.ndarray) and got.dtype == np.float32
    _check(torch.from_numpy(got), dict(c, x=torch.from_numpy(xf), y=torch.from_numpy(plain)))
    dev = proj.apply(torch.from_numpy(xf).to(gpu), adapters=ad, index=index)
    assert torch.equal(dev.cpu(), torch.from_numpy(got))
    with pytest.raises(ValueError):
        proj.apply(xf, adapters=ad)


def on_norm(x, w, res):
    s = (x.float() + res.float()).double()
    return s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()


@pytest.mark.parametrize("T", [300, 600, 1111, 4500])
def test_views_of_many_rows(gpu, T):
    """Rows at odd offsets and strides for every number of tokens, K a multiple
    of 8 and not, with guards around y."""
    from ccut.quant import lora

    for K, N, off, R, t in ((96, 77, 1, 16, "bf16"), (256, 264, 8, 40, "f16"), (100, 64, 3, 130, "bf16"),
                            (64, 72, 1, 8, "f32")):
        c = _case(T, K, N, R, 4, t, "bf16" if t == "f32" else t, t, ranks=True)
        big = torch.full((T + 2, K + N + 20), 5.0, dtype=DT[t], device=gpu)
        xs, ys = big[1:-1, off:off + K], big[1:-1, off + K:off + K + N]
        xs.copy_(c["x"].to(gpu))
        ys.copy_(c["y"].to(gpu))
        before = big.clone()
        lora.add_(ys, xs, _adapters(c, gpu), c["index"].to(gpu))
        _check(ys, c)
        ys.copy_(c["y"].to(gpu))
        assert torch.equal(big, before)


def test_smallest_buffers_many_tokens(gpu):
    """Adapters of a few values beside many tokens, long rows or wide ones."""
    for T, K, N, R, L in ((65536, 40, 1, 1, 1), (4100, 2000, 7, 1, 1), (3000, 1, 700, 7, 1), (4, 1, 3000, 256, 5),
                          (1, 7, 100, 200, 3)):
        for t in ("bf16", "f32"):
            c = _case(T, K, N, R, L, t, "bf16", t)
            _check(_run(c, gpu), c)


def test_far_inputs(gpu):
    """Rows of x beyond 2^32 bytes, for the tiles of few and of many tokens."""
    from ccut.quant import lora

    buf = torch.empty(36000 * 65536 + 64, dtype=torch.bfloat16, device=gpu)
    for T, ld in ((36000, 65536), (300, 7864320)):
        c = _case(T, 64, 40, 8, 3, "bf16", "bf16", "bf16")
        xs = buf[8:8 + T * ld].view(T, ld)[:, :64]
        assert (T - 1) * ld * 2 > 2 ** 32
        xs.copy_(c["x"].to(gpu))
        y = c["y"].to(gpu)
        lora.add_(y, xs, _adapters(c, gpu), c["index"].to(gpu))
        _check(y, c)


@pytest.mark.parametrize("T", [6, 200, 900])
def test_one_stack_on_two_streams(gpu, T):
    """The same adapters, rows and index in calls that run at once."""
    from ccut.quant import lora

    c = _case(T, 640, 300, 24, 5, "bf16", "bf16", "bf16")
    ad, x, index = _adapters(c, gpu), c["x"].to(gpu), c["index"].to(gpu)
    want = _run(c, gpu)
    _check(want, c)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        ys = [c["y"].to(gpu) for _ in range(6)]
        torch.cuda.synchronize()
        for n, y in enumerate(ys):
            with torch.cuda.stream(streams[n & 1]):
                lora.add_(y, x, ad, index)
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in ys), f"turn {turn}"


@pytest.mark.parametrize("T", [1, 48, 700])
def test_captured_chain(gpu, T):
    """Norm, 8-bit projection and adapters in one graph, the residual in
    place, replayed on new rows with eager work between."""
    from ccut import workloads
    from ccut.blocks import norm
    from ccut.quant import fp8_block, lora

    H, N, R, L = 512, 384, 16, 4
    g = torch.Generator(device=gpu).manual_seed(T)
    w = 1 + 0.1 * torch.randn(H, generator=g, device=gpu)
    wq, ws = workloads.fp8_block_weights(1, N, H, 1, gpu)
    lin = fp8_block.prepare(wq[0], ws[0], H)
    c = _case(T, H, N, R, L, "bf16", "bf16", "bf16")
    ad = _adapters(c, gpu)

    def layer(x, res, index):
        q, scale, y, _ = norm.rms_norm_fp8(x, w, residual=res, residual_out=res, normed=True)
        return lora.add_(fp8_block.linear_quantized(lin, q, scale), y, ad, index)

    rows = [[torch.randn((T, H), generator=g, device=gpu).bfloat16() for _ in range(2)] +
            [torch.randint(-1, L, (T,), generator=g, device=gpu)] for _ in range(3)]
    held = [t.clone() for t in rows[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(*held)
    for n in (1, 0, 2, 1):
        for to, src in zip(held, rows[n]):
            to.copy_(src)
        graph.replay()
        again = [t.clone() for t in rows[n]]
        want = layer(*again)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(held[1], again[1]), f"rows {n}"


def test_rows_quantized_already_refusals(gpu):
    from ccut import workloads
    from ccut.quant import fp8_block

    wq, ws = workloads.fp8_block_weights(1, 128, 256, 1, gpu)
    lin = fp8_block.prepare(wq[0], ws[0], 256)
    q, s = torch.zeros((3, 256), dtype=torch.uint8, device=gpu), torch.ones((3, 2), device=gpu)
    for f in (lambda: fp8_block.linear_quantized(lin, q.float(), s), lambda: fp8_block.linear_quantized(lin, q, s.half()),
              lambda: fp8_block.linear_quantized(lin, q[:, :128], s), lambda: fp8_block.linear_quantized(lin, q, s[:2]),
              lambda: fp8_block.linear_quantized(lin, q, s[:, :1]), lambda: fp8_block.linear_quantized(lin, q.cpu(), s),
              lambda: fp8_block.linear_quantized(lin, q, s.cpu()),
              lambda: fp8_block.linear_quantized(lin, q, s, torch.float64)):
        with pytest.raises(ValueError):
            f()
    assert fp8_block.linear_quantized(lin, q[:0], s[:0]).shape == (0, 128)
    big = torch.randint(0, 100, (7, 300), dtype=torch.uint8, device=gpu)  # codes at an odd address and stride
    got = fp8_block.linear_quantized(lin, big[:, 3:259], torch.ones((7, 2), device=gpu), torch.float32)
    want = fp8_block.linear_quantized(lin, big[:, 3:259].clone(), torch.ones((7, 2), device=gpu), torch.float32)
    assert torch.equal(got, want)
    one = fp8_block.linear_quantized(lin, big[0, 3:259].view(torch.float8_e4m3fn), torch.ones(2, device=gpu),
                                     torch.float32)
    assert one.shape == (128,)


@pytest.mark.parametrize("T,K,R,L", [(2048, 4096, 16, 8), (4096, 2048, 128, 6), (1500, 3600, 40, 20)])
@pytest.mark.parametrize("pattern", ["one", "runs", "mixed", "none"])
def test_splits_by_the_number_of_tiles(gpu, T, K, R, L, pattern):
    """Tiles without padding, with some, with as much as there can be, and none."""
    for types in (("bf16", "bf16", "bf16"), ("f32", "f16", "f32")):
        c = _case(T, K, 40, R, L, *types, pattern=pattern)
        _check(_run(c, gpu), c)


def _factor(c, f):
    """The adapters' products times f, and y with them."""
    c["scale"] = torch.where(torch.arange(c["a"].shape[0]) % 2 == 0, 1.0, -0.75) * f
    c["y"] = (c["y"].double() * f).to(c["y"].dtype)
    return c


@pytest.mark.parametrize("power", [110, 116, 120, 122, -100, -108, -114, -120])
@pytest.mark.parametrize("T,K,R", [(5, 64, 16), (40, 200, 40), (600, 72, 24), (600, 75, 130)])
def test_products_over_the_float32_range(gpu, T, K, R, power):
    """Scaled inner products near both ends of float32's range.  (Parts in
    bfloat16 end at 2^-133: products below 2^-107 keep fewer bits there.)"""
    for types in (("f32", "f16", "f32"), ("f16", "f16", "f32"), ("f32", "bf16", "f32"), ("bf16", "bf16", "f32")):
        if types[1] == "bf16" and power < -100:
            continue
        c = _factor(_case(T, K, 72, R, 3, *types), 2.0 ** power)
        _check(_run(c, gpu), c)


@pytest.mark.parametrize("T,R", [(5, 16), (40, 40), (600, 24)])
def test_largest_products(gpu, T, R):
    """Inner products that round to infinity in bfloat16 and are finite in
    float32: 2^127 (2 - 2^-8) and more."""
    for ydt in ("f32", "bf16"):
        c = _case(T, 64, 72, R, 2, "f32", "bf16", ydt, scale=False)
        c["x"].zero_()
        c["x"][:, 3] = torch.where(torch.arange(T) % 3 == 0, -1.0, 1.0) * torch.linspace(3.3896e38, 3.4028e38, T)
        c["a"].zero_()
        c["a"][:, ::5, 3] = 1.0
        c["b"] = torch.zeros_like(c["b"])
        c["b"][:, :, 0] = torch.linspace(-0.75, 0.75, 72).bfloat16()  # 0 among them
        c["b"][:, 36, 0] = 0.0
        _check(_run(c, gpu), c)


def test_projection_with_adapters_takes_what_it_takes_without(gpu):
    """Rows of any type that ``apply`` converts, an index of any whole
    numbers; one that would be cut to whole numbers is refused."""
    from ccut.quant.linear import FakeWeightReader, LinearProj

    T, K, N = 9, 64, 48
    c = _case(T, K, N, 8, 3, "f32", "bf16", "f32")
    ad = _adapters(c, gpu)
    rng = np.random.default_rng(1)
    wf = rng.standard_normal((N, K)).astype(np.float32)
    proj = LinearProj(0, "proj", N, K, FakeWeightReader({(0, "proj"): wf.tobytes()}, {(0, "proj"): (N, K, "F32")}), None)
    for x in (c["x"].to(gpu), c["x"].to(gpu).double(), c["x"].numpy().astype(np.float64),
              torch.randint(-4, 5, (T, K), device=gpu)):
        plain = torch.as_tensor(proj.apply(x)).cpu()
        want = dict(c, x=torch.as_tensor(x).cpu().float(), y=plain)
        for index in (c["index"].to(gpu), c["index"].tolist(), c["index"].numpy().astype(np.int16)):
            _check(torch.as_tensor(proj.apply(x, adapters=ad, index=index)), want)
    for index in (c["index"].numpy().astype(np.float32), c["index"].to(gpu).double(), c["index"].numpy() >= 0):
        with pytest.raises(ValueError, match="whole numbers"):
            proj.apply(c["x"].numpy(), adapters=ad, index=index)
    none = np.zeros((0, K), np.float32)
    assert proj.apply(none).shape == proj.apply(none, adapters=ad, index=[]).shape == (0, N)


@pytest.mark.parametrize("K", [2048, 4104, 3601])
@pytest.mark.parametrize("T", [4097, 5000, 8192])
def test_splits_above_the_self_sorted_batches(gpu, T, K):
    """K in several parts behind the schedule's own launch: whole and partial
    last stages, rows that are not aligned, few and many tiles (5000 tokens of
    40 adapters take another number of parts for each)."""
    for R, L, pattern, types in ((16, 3, "runs", ("bf16", "bf16", "bf16")), (64, 40, "one", ("f16", "f16", "f16")),
                                 (64, 40, "mixed", ("f16", "f16", "f32")), (128, 7, "runs", ("f32", "bf16", "f32")),
                                 (200, 40, "runs", ("bf16", "bf16", "f32")), (32, 40, "one", ("f32", "f16", "f32")),
                                 (16, 5, "none", ("bf16", "bf16", "bf16"))):
        c = _case(T, K, 40, R, L, *types, pattern=pattern, ranks=R == 64 and pattern == "mixed")
        _check(_run(c, gpu), c)


def test_far_inputs_of_one_copy_base(gpu):
    """Rows of x between 2^31 and 2^32 bytes behind the first, as 32-bit
    offsets of aligned copies, for tiles of few tokens in one kernel and of
    many.  x begins 2^31 bytes into its buffer, which holds any such offset."""
    from ccut.quant import lora

    buf = torch.empty(3 * 2 ** 30 + 2 ** 22, dtype=torch.bfloat16, device=gpu)
    for T, ld in ((16, 130000000), (700, 2900000), (5000, 420000)):
        c = _case(T, 128, 40, 16, 3, "bf16", "bf16", "bf16")
        assert 2 ** 31 < (T - 1) * ld * 2 and (ld + 1) * T * 2 <= 2 ** 32 and ld % 8 == 0
        xs = buf[2 ** 30:2 ** 30 + T * ld].view(T, ld)[:, :128]
        xs.copy_(c["x"].to(gpu))
        y = c["y"].to(gpu)
        lora.add_(y, xs, _adapters(c, gpu), c["index"].to(gpu))
        _check(y, c)


@pytest.mark.parametrize("types", TYPES, ids="-".join)
@pytest.mark.parametrize("T,K,R", [(5, 64, 16), (70, 128, 32), (90, 200, 40), (600, 72, 24), (600, 75, 130)])
def test_infinite_weights(gpu, T, K, R, types):
    """Infinities in b give what the whole products give: infinities of the
    product's sign, NaN only where two of them differ or the product is 0."""
    c = _case(T, K, 200, R, 3, *types)
    c["x"][1] = 0.0
    c["index"][1] = 2
    for i, n, r, v in ((0, 0, 0, "inf"), (0, 69, R - 1, "-inf"), (2, 7, 3, "inf"), (2, 7, 8, "inf"), (2, 199, 1, "-inf")):
        c["b"][i, n, r] = float(v)
    y = _run(c, gpu).cpu()
    ref, bound = ol.add(c["y"], c["x"], c["a"], c["b"], c["index"], c["scale"], c["rank"])
    fine = torch.isfinite(ref)
    off, tol = (y.double() - ref).abs(), bound(c["y"].dtype, c["a"].dtype)
    assert (off[fine] <= tol[fine]).all(), f"worst {(off / tol)[fine].max():.3f} of the bound"
    assert torch.equal(y.isnan(), ref.isnan())
    assert torch.equal(y[ref.isinf()].double(), ref[ref.isinf()])
    assert ref.isinf().any() and ref[1].isnan().any()


def test_stacks_are_not_exchanged(gpu):
    """Another tensor in the place of a stack is refused (the calls would read
    the old one); the memory that the calls read lives as long as the handle."""
    from ccut.quant import lora

    c = _case(30, 128, 96, 16, 3, "bf16", "bf16", "bf16", ranks=True)
    ad = _adapters(c, gpu)
    for name in ("a", "b", "scale", "rank", "in_features"):
        with pytest.raises(AttributeError, match="writing into"):
            setattr(ad, name, getattr(ad, name))
    ad.label = "q_proj"
    ad.label = "k_proj"
    kept = [t.clone() for t in (ad.a, ad.b)]
    ad.a.data, ad.b.data = torch.zeros_like(kept[0]), torch.zeros_like(kept[1])  # their old memory is not handed out
    for _ in range(4):
        torch.full_like(kept[0], float("nan")), torch.full_like(kept[1], float("nan"))
    _check(lora.add_(c["y"].to(gpu), c["x"].to(gpu), ad, c["index"].to(gpu)), c)


def test_captured_above_the_self_sorted_batches(gpu):
    """A captured call of more than 4096 tokens, K in parts, replayed on other
    rows and other numbers of tiles with eager work between the replays."""
    from ccut.quant import lora

    T, K, N, R, L = 5000, 2048, 72, 24, 40
    cs = [_case(T, K, N, R, L, "bf16", "bf16", "bf16", seed=s, pattern=p) for s, p in
          enumerate(("one", "mixed", "none", "runs"))]
    ad = _adapters(cs[0], gpu)
    x, y, index = (cs[0][k].to(gpu) for k in ("x", "y", "index"))
    lora.add_(y, x, ad, index)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lora.add_(y, x, ad, index)
    for n in (1, 0, 3, 2, 0):
        for to, k in ((x, "x"), (y, "y"), (index, "index")):
            to.copy_(cs[n][k].to(gpu))
        graph.replay()
        want = lora.add_(cs[n]["y"].to(gpu), cs[n]["x"].to(gpu), ad, cs[n]["index"].to(gpu))
        torch.cuda.synchronize()
        assert torch.equal(y, want), f"rows {n}"
        _check(y, dict(cs[n], a=cs[0]["a"], b=cs[0]["b"], scale=cs[0]["scale"]))
