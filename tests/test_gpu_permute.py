"""Tokens sorted by expert and back (``ccq_moe_permute``,
``ccq_moe_unpermute``, ``ccq_moe_unpermute_grad``), their gradients, and the
layer of 16-bit experts built of them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import dense as od
from oracle import permute as op

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _ids(T, k, E, seed=0, bare=0.1, skew=1.0):
    g = torch.Generator().manual_seed(seed * 31 + T + 7 * k + E)
    score = torch.rand((T, E), generator=g) + skew * torch.rand(E, generator=g)
    ids = score.argsort(1, descending=True)[:, :k].clone()
    ids[torch.rand((T, k), generator=g) < bare] = -1
    return ids


def _close(y, ref, tol):
    assert torch.isfinite(y).all()
    off = (y.cpu().double() - ref).abs()
    assert (off <= tol).all(), f"worst {(off / tol.clamp_min(1e-300)).max():.3f} of the bound"


def _check(gpu, ids, E, H, dt, seed=0):
    from ccut.blocks import moe

    T, k = ids.shape
    g = torch.Generator().manual_seed(seed + T + H)
    x, dy = (torch.randn((T, H), generator=g).to(dt) for _ in range(2))
    rows = torch.randn((T * k, H), generator=g).to(dt)
    w = torch.randn((T, k), generator=g)
    position, offsets = op.plan(ids, E)
    got, plan = moe.moe_permute(x.to(gpu), ids.to(gpu), E)
    assert torch.equal(plan.position.cpu(), position) and torch.equal(plan.offsets.cpu(), offsets)
    assert torch.equal(got.cpu(), op.permute(x, position))
    y, bound = op.unpermute(rows, position, w)
    for ydt in {dt, F32}:
        _close(moe.moe_unpermute(rows.to(gpu), plan, w.to(gpu), ydt), y, bound(ydt))
    y, bound = op.unpermute(rows, position)
    _close(moe.moe_permute_backward(rows.to(gpu), plan), y, bound(dt))
    d_rows, d_w = moe.moe_unpermute_backward(dy.to(gpu), rows.to(gpu), plan, w.to(gpu))
    ref, ref_w, tol_w = op.unpermute_backward(dy, rows, position, w)
    f = torch.finfo(dt)  # one product, rounded to float32 and to the type
    _close(d_rows, ref, ref.abs() * (f.eps / 2 + 2.0 ** -24) * 1.01 + f.smallest_normal * f.eps)
    _close(d_w, ref_w, tol_w)


@pytest.mark.parametrize("dt", [BF, F16, F32])
@pytest.mark.parametrize("T,k,E,H", [(1, 1, 1, 64), (1, 8, 128, 2048), (16, 6, 64, 256), (37, 3, 5, 130), (500, 8, 16, 512),
                                     (512, 8, 40, 64), (513, 8, 40, 64), (1025, 4, 256, 72), (2000, 4, 4, 64),
                                     (700, 8, 1024, 40)])
def test_types_and_batches(gpu, T, k, E, H, dt):
    _check(gpu, _ids(T, k, E), E, H, dt)


@pytest.mark.parametrize("H", [1, 2, 3, 4, 5, 7, 8, 9, 15, 17, 31, 33, 63, 65, 127, 129, 255, 257, 509, 1000, 2047, 4099,
                               7168, 9001])
def test_row_lengths(gpu, H):
    for dt in (BF, F32):
        _check(gpu, _ids(9, 3, 6), 6, H, dt)
        _check(gpu, _ids(1030, 2, 6), 6, min(H, 600), dt)


@pytest.mark.parametrize("k", [1, 2, 7, 8, 9, 15, 16, 17, 33, 64])
def test_slots(gpu, k):
    for T in (3, 130):
        _check(gpu, _ids(T, k, 70), 70, 96, BF)


def test_long_batches(gpu):
    """Counts in chunks: whole and ragged ones, the most assignments."""
    for T, k, E, H in ((4096, 8, 128, 16), (4097, 7, 60, 8), (8192, 8, 256, 8), (131072, 8, 300, 1), (16384, 64, 1024, 1)):
        from ccut.blocks import moe

        ids = torch.randint(-1, E, (T, k), generator=torch.Generator().manual_seed(T))
        x = torch.arange(T, dtype=F32)[:, None].expand(T, H).contiguous()
        rows, plan = moe.moe_permute(x.to(gpu), ids.to(gpu), E)
        key = torch.where(ids.view(-1) < 0, E, ids.view(-1))
        order = torch.sort(key, stable=True).indices
        at = torch.empty(T * k, dtype=torch.int64)
        at[order] = torch.arange(T * k)
        assert torch.equal(plan.position.cpu().view(-1).long(), torch.where(key == E, ~at, at))
        counts = torch.bincount(key, minlength=E + 1)[:E].cumsum(0)
        assert plan.offsets[0] == 0 and torch.equal(plan.offsets.cpu()[1:].long(), counts)
        kept = int(counts[-1])
        assert torch.equal(rows.cpu()[:kept, -1], (order // k)[:kept].float()) and (rows[kept:] == 0).all()


@pytest.mark.parametrize("pattern", ["one", "none", "twice", "beyond", "last"])
@pytest.mark.parametrize("T", [1, 5, 300, 1500])
def test_patterns(gpu, T, pattern):
    E, k = 9, 4
    ids = {"one": torch.full((T, k), 3), "none": torch.full((T, k), -1),
           "twice": torch.tensor([5, 5, 0, 5]).expand(T, k).clone(),
           "beyond": torch.randint(-4, 14, (T, k), generator=torch.Generator().manual_seed(T)),
           "last": torch.full((T, k), E - 1)}[pattern]
    if pattern == "beyond":
        ids[0, 0], ids[-1, -1] = 2 ** 40, -2 ** 62
    _check(gpu, ids, E, 40, BF)


def test_strides_types_of_ids_and_empty(gpu):
    from ccut.blocks import moe

    ids = _ids(20, 3, 6)
    position, offsets = op.plan(ids, 6)
    for shift in range(9):
        buf = torch.randn(20 * 45 + 16, device=gpu).to(BF)
        x = buf[shift:shift + 20 * 45].view(20, 45)[:, :36]
        rows, plan = moe.moe_permute(x, ids.to(gpu).int() if shift % 2 else ids.to(gpu).t().contiguous().t(), 6)
        assert torch.equal(rows.cpu(), op.permute(x.cpu(), position)) and torch.equal(plan.offsets.cpu(), offsets)
        wide = torch.randn(60 * 45 + 16, device=gpu).to(BF)[shift:shift + 60 * 45].view(60, 45)[:, 3:39]
        y, bound = op.unpermute(wide.cpu(), position)
        _close(moe.moe_unpermute(wide, plan), y, bound(BF))
        w = torch.rand((20, 3))
        d_rows, d_w = moe.moe_unpermute_backward(x, wide, plan, w.to(gpu))
        ref, ref_w, tol = op.unpermute_backward(x.cpu(), wide.cpu(), position, w)
        _close(d_rows, ref, ref.abs() * (2.0 ** -8 + 2.0 ** -23) + 1e-39)
        _close(d_w, ref_w, tol)
    # gradients as autograd hands them over: one row for all
    dy = torch.randn(36, device=gpu).to(BF).expand(20, 36)
    d_rows, _ = moe.moe_unpermute_backward(dy, wide, plan, w.to(gpu))
    ref, _, _ = op.unpermute_backward(dy.cpu(), wide.cpu(), position, w)
    _close(d_rows, ref, ref.abs() * (2.0 ** -8 + 2.0 ** -23) + 1e-39)
    rows, plan = moe.moe_permute(torch.zeros((0, 8), device=gpu), torch.zeros((0, 2), dtype=torch.int64, device=gpu), 5)
    assert rows.shape == (0, 8) and plan.position.shape == (0, 2) and (plan.offsets == 0).all() and plan.offsets.numel() == 6
    assert moe.moe_unpermute(rows, plan).shape == (0, 8)


def test_not_finite_in_left_out_rows(gpu):
    """What stands in rows of left-out assignments is not read, whatever their weights."""
    from ccut.blocks import moe

    ids = _ids(40, 4, 6, bare=0.3)
    ids[3] = -1
    position, offsets = op.plan(ids, 6)
    plan = moe.Permutation(position.to(gpu), offsets.to(gpu))
    rows, w = torch.randn((160, 33)), torch.rand((40, 4))
    rows[int(offsets[-1]):] = float("nan")
    w[ids < 0] = float("inf")
    clean = torch.where(ids < 0, 0.0, w)
    y, bound = op.unpermute(rows, position, clean)
    got = moe.moe_unpermute(rows.to(gpu), plan, w.to(gpu))
    _close(got, y, bound(F32))
    assert (got[3] == 0).all()
    dy = torch.randn((40, 33))
    d_rows, d_w = moe.moe_unpermute_backward(dy.to(gpu), rows.to(gpu), plan, w.to(gpu))
    ref, ref_w, tol = op.unpermute_backward(dy, rows, position, clean)
    _close(d_rows, ref, ref.abs() * 2.0 ** -23 + 1e-40)
    _close(d_w, ref_w, tol)
    # an infinity in a kept row is its token's alone
    rows[0, 5] = float("inf")
    owner = int((position == 0).nonzero()[0, 0])
    got = moe.moe_unpermute(rows.to(gpu), plan, w.to(gpu)).cpu()
    assert got[owner, 5] == float("inf") and torch.isfinite(got).sum() == got.numel() - 1


def test_gradients_against_differences(gpu):
    """Both functions are linear in each argument: central differences are exact but for rounding."""
    from ccut.blocks import moe

    T, k, E, H = 30, 3, 7, 50
    g = torch.Generator().manual_seed(3)
    ids = _ids(T, k, E).to(gpu)
    rnd = lambda *s: torch.randn(s, generator=g).to(gpu)  # noqa: E731
    x, d_out, step_x = rnd(T, H), rnd(T * k, H), rnd(T, H)
    rows, plan = moe.moe_permute(x, ids, E)
    up, down = moe.moe_permute(x + step_x, ids, E)[0], moe.moe_permute(x - step_x, ids, E)[0]
    num = ((up.double() - down.double()) / 2 * d_out.double()).sum()
    ana = (moe.moe_permute_backward(d_out, plan).double() * step_x.double()).sum()
    size = (d_out.abs().double().sum() * 4)
    assert abs(num - ana) <= 16 * 2.0 ** -24 * size
    w, dy, step_r, step_w = rnd(T, k), rnd(T, H), rnd(T * k, H), rnd(T, k)
    d_rows, d_w = moe.moe_unpermute_backward(dy, rows, plan, w)
    f = lambda r, v: (moe.moe_unpermute(r, plan, v).double() * dy.double()).sum()  # noqa: E731
    size = 4 * (dy.abs().double().sum() * k * 16)
    assert abs((f(rows + step_r, w) - f(rows - step_r, w)) / 2 - (d_rows.double() * step_r.double()).sum()) <= (
        16 * 2.0 ** -24 * size)
    assert abs((f(rows, w + step_w) - f(rows, w - step_w)) / 2 - (d_w.double() * step_w.double()).sum()) <= (
        16 * 2.0 ** -24 * size)


def _layer(E, H, I, dt, seed=0):
    g = torch.Generator().manual_seed(seed + E + H)
    return ((torch.randn((E, 2 * I, H), generator=g) * H ** -0.5).to(dt), (torch.randn((E, H, I), generator=g) * I ** -0.5).to(dt),
            torch.randn((E, 2 * I), generator=g).to(dt), torch.randn((E, H), generator=g))


def _layer_ref(x, ids, weights, E, wgu, wd, bgu, bd, act, ydt):
    """The layer in 64 bits, and the bound: each step's own plus what the steps before hand on."""
    dt = x.dtype
    position, offsets = op.plan(ids, E)
    rows = op.permute(x, position)
    h, bh = od.grouped(rows, offsets, wgu, bgu, act, True)
    eh = bh(dt)
    d, bd_ = torch.zeros((rows.shape[0], wd.shape[1]), dtype=torch.float64), None
    ed = torch.zeros_like(d)
    for e in range(E):
        b, n = int(offsets[e]), int(offsets[e + 1])
        if n > b:
            y, bound = od.linear(h[b:n], wd[e], bd[e] if bd is not None else None)
            d[b:n] = y
            # the inputs differ from h by eh: their products, and the bound's own growth
            carried = eh[b:n] @ wd[e].double().abs().t()
            ed[b:n] = bound(dt) + carried * (1 + torch.finfo(dt).eps + wd.shape[2] * 2.0 ** -24)
    y, bound = op.unpermute(d, position, weights)
    e, _ = op.unpermute(ed, position, weights.abs())
    return y, bound(ydt) + e * (1 + torch.finfo(ydt).eps + 1e-5)


@pytest.mark.parametrize("T,k,E,H,I", [(1, 8, 16, 256, 96), (40, 6, 64, 128, 72), (600, 4, 8, 192, 130), (1100, 8, 12, 64, 64)])
@pytest.mark.parametrize("dt,bias,act", [(BF, False, "silu"), (F16, True, "gelu")])
def test_layer_of_dense_experts(gpu, T, k, E, H, I, dt, bias, act):
    from ccut.blocks import moe

    wgu, wd, bgu, bd = _layer(E, H, I, dt)
    if not bias:
        bgu = bd = None
    g = torch.Generator().manual_seed(T)
    x, w = torch.randn((T, H), generator=g).to(dt), torch.rand((T, k), generator=g)
    ids = _ids(T, k, E)
    up = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    ex = moe.DenseExperts(up(wgu), up(wd), up(bgu), up(bd), act=act)
    for ydt in (dt, F32):
        y, tol = _layer_ref(x, ids, w, E, wgu, wd, bgu, bd, act, ydt)
        _close(moe.moe_ffn_dense(x.to(gpu), ids.to(gpu), w.to(gpu), ex, ydt), y, tol)
    shared = torch.randn((T, H), generator=g)
    got = moe.moe_ffn_dense(x.to(gpu), ids.to(gpu), w.to(gpu), ex, F32, shared=shared.to(gpu), shared_gate=0.5)
    y, tol = _layer_ref(x, ids, w, E, wgu, wd, bgu, bd, act, F32)
    y = y + 0.5 * shared.double()
    _close(got, y, tol + 2.0 ** -23 * (y.abs() + shared.abs()))


def test_forward_dense_and_pipeline(gpu):
    """The layer from router logits, and as a reader's experts in ExpertPipeline.step."""
    from ccut.blocks import moe
    from ccut.experts.pipeline import ExpertPipeline

    T, k, E, H, I = 24, 4, 16, 128, 64
    wgu, wd, _, _ = _layer(E, H, I, BF)
    ex = moe.DenseExperts.from_stacks(wgu[:, :I], wgu[:, I:], wd)
    assert torch.equal(ex.w_gate_up.cpu(), wgu) and (ex.num_experts, ex.hidden, ex.inter) == (E, H, I)
    g = torch.Generator().manual_seed(1)
    x, lg = torch.randn((T, H), generator=g).to(BF), torch.randn((T, E), generator=g)
    w, ids = moe.topk_softmax(lg.to(gpu), k)
    y, tol = _layer_ref(x, ids.cpu(), w.cpu(), E, wgu, wd, None, None, "silu", BF)
    _close(moe.moe_forward_dense(x.to(gpu), lg.to(gpu), ex, k), y, tol)

    class Reader:
        def experts(self, layer):
            return ex

    gate = torch.randn((E, H), generator=g)
    pipe = ExpertPipeline(Reader())
    xs = x.float()  # float32 rows that bfloat16 holds exactly
    out = pipe.step(0, xs.numpy(), gate.numpy(), top_k=k)
    w, ids = moe.topk_softmax(pipe.router_logits(xs.to(gpu), gate.to(gpu)), k)
    y, tol = _layer_ref(x, ids.cpu(), w.cpu(), E, wgu, wd, None, None, "silu", F32)
    assert isinstance(out, np.ndarray) and out.dtype == np.float32
    _close(torch.from_numpy(out), y, tol)


def test_graphs(gpu):
    """The layer captured, for a batch that one workgroup's comparisons sort and one counted in chunks; replays
    with eager work between them against eager results."""
    from ccut.blocks import moe

    E, H, I, k = 12, 64, 48, 8
    wgu, wd, _, _ = _layer(E, H, I, BF)
    ex = moe.DenseExperts(wgu.to(gpu), wd.to(gpu))
    gen = torch.Generator().manual_seed(9)
    state = []
    for T in (20, 700, 900):
        x, w, ids = torch.randn((T, H), device=gpu).to(BF), torch.rand((T, k), device=gpu), _ids(T, k, E).to(gpu)
        dy = torch.randn((T, H), device=gpu).to(BF)

        def call(x=x, w=w, ids=ids, dy=dy):
            rows, plan = moe.moe_permute(x, ids, E)
            return (moe.moe_ffn_dense(x, ids, w, ex), plan.offsets, *moe.moe_unpermute_backward(dy, rows, plan, w),
                    moe.moe_permute_backward(rows, plan))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = call()
        state.append((g, outs, call, x, w, ids))
    for i in range(4):
        want = []
        for g, outs, call, x, w, ids in state:
            x.copy_(torch.randn(x.shape, generator=gen))
            ids.copy_(_ids(*ids.shape, E, seed=i + 1))
            want.append(call())
        for g, *_ in state:
            g.replay()
        torch.cuda.synchronize()
        for (g, outs, *_), ys in zip(state, want):
            for o, y in zip(outs, ys):
                assert torch.equal(o, y)


@pytest.mark.parametrize("T,k,H", [(1 << 17, 8, 8200), (1 << 20, 1, 8200)])
def test_rows_beyond_32_bits(gpu, T, k, H):
    """Rows that take 16 GiB, there and back; the second has more pieces than a row of the grid."""
    from ccut.blocks import moe

    E = 40
    g = torch.Generator(device=gpu).manual_seed(T)
    x = torch.randint(-4, 5, (T, 1), generator=g, device=gpu).to(BF) + torch.arange(H, device=gpu).remainder(3).to(BF)
    ids = torch.randint(0, E, (T, k), generator=g, device=gpu)
    rows, plan = moe.moe_permute(x, ids, E)
    at = torch.empty(T * k, dtype=torch.int64, device=gpu)
    at[torch.sort(ids.view(-1), stable=True).indices] = torch.arange(T * k, device=gpu)
    assert torch.equal(plan.position.view(-1).long(), at)
    for s in range(k):
        at = plan.position[:, s].long()
        for t in range(0, T, 1 << 17):
            assert torch.equal(rows[at[t:t + (1 << 17)]], x[t:t + (1 << 17)])
    y = moe.moe_permute_backward(rows, plan)
    for t in range(0, T, 1 << 17):  # (small whole numbers: exact)
        assert torch.equal(y[t:t + (1 << 17)], x[t:t + (1 << 17)] * k)
    del y
    w = torch.ones((T, k), device=gpu)
    d_rows, d_w = moe.moe_unpermute_backward(x, rows, plan, w)
    for t in range(0, T * k, 1 << 17):
        assert torch.equal(d_rows[t:t + (1 << 17)], rows[t:t + (1 << 17)])
    some = torch.cat([torch.arange(5), torch.arange(T - 5, T)]).to(gpu)
    assert torch.equal(d_w[some].cpu(), x[some].double().square().sum(1).float().cpu()[:, None].expand(-1, k))
    del rows, d_rows, x
    torch.cuda.empty_cache()


def test_refusals(gpu):
    from ccut.blocks import moe

    x, ids = torch.zeros((6, 16), device=gpu), torch.zeros((6, 2), dtype=torch.int64, device=gpu)
    rows, plan = moe.moe_permute(x, ids, 3)
    w = torch.zeros((6, 2), device=gpu)
    bad = moe.Permutation(plan.position.long(), plan.offsets)
    short = moe.Permutation(plan.position[:5], plan.offsets)
    ex = moe.DenseExperts(torch.zeros((3, 16, 16), dtype=BF, device=gpu), torch.zeros((3, 16, 8), dtype=BF, device=gpu))
    for call in (lambda: moe.moe_permute(x.cpu(), ids, 3), lambda: moe.moe_permute(x, ids.cpu(), 3),
                 lambda: moe.moe_permute(x.double(), ids, 3), lambda: moe.moe_permute(x, ids[:5], 3),
                 lambda: moe.moe_permute(x, ids.float(), 3), lambda: moe.moe_permute(x, ids, 0),
                 lambda: moe.moe_permute(x, ids, 1025), lambda: moe.moe_permute(x, ids[:, :0], 3),
                 lambda: moe.moe_permute(x, torch.zeros((6, 65), dtype=torch.int64, device=gpu), 3),
                 lambda: moe.moe_permute(x[0], ids, 3), lambda: moe.moe_unpermute(rows.cpu(), plan),
                 lambda: moe.moe_unpermute(rows[:-1], plan), lambda: moe.moe_unpermute(rows, bad),
                 lambda: moe.moe_unpermute(rows, short), lambda: moe.moe_unpermute(rows, plan, w[:, :1]),
                 lambda: moe.moe_unpermute(rows, plan, w.long()), lambda: moe.moe_unpermute(rows, plan, w.cpu()),
                 lambda: moe.moe_unpermute(rows, plan, out_dtype=torch.float64),
                 lambda: moe.moe_unpermute_backward(x.half(), rows, plan, w),
                 lambda: moe.moe_unpermute_backward(x[:5], rows, plan, w),
                 lambda: moe.moe_unpermute_backward(x, rows[:-2], plan, w),
                 lambda: moe.moe_unpermute_backward(x, rows, plan, w[:3]),
                 lambda: moe.moe_unpermute_backward(x, rows, plan, None),
                 lambda: moe.moe_ffn_dense(x, ids, w, ex), lambda: moe.moe_ffn_dense(x.to(BF)[:, :8], ids, w, ex),
                 lambda: moe.DenseExperts(ex.w_gate_up, ex.w_down.half()),
                 lambda: moe.DenseExperts(ex.w_gate_up[:, :8], ex.w_down),
                 lambda: moe.DenseExperts(ex.w_gate_up, ex.w_down, act="tanh"),
                 lambda: moe.DenseExperts(ex.w_gate_up, ex.w_down, torch.zeros(3, 8))):
        with pytest.raises(ValueError):
            call()
