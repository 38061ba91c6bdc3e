"""ccq_dense_linear(_grouped), ccq_moe_permute, ccq_moe_unpermute and
ccq_moe_unpermute_grad refuse bad arguments on the host before anything is
launched, the Python entry points refuse host tensors, and the oracle of the
gradients agrees with differences (runs without a GPU)."""

from __future__ import annotations

import pytest
import torch

P = 256  # an address that is never used: validation comes first


@pytest.fixture(scope="module")
def lib(built_lib):
    from ccut import _lib

    return _lib.lib()


FIELDS = ("x", "w", "bias", "residual", "y", "offsets", "workspace", "stream", "workspace_bytes", "ldx", "ldr", "ldy", "M",
          "K", "N", "num_experts", "dtype", "bias_dtype", "y_dtype", "act", "gated")


def _args(**kw):
    from ccut._lib import DENSE_ARGS

    a = dict(x=P, w=P, bias=0, residual=0, y=P, offsets=P, workspace=0, stream=0, workspace_bytes=0, ldx=64, ldr=32, ldy=32,
             M=4, K=64, N=32, num_experts=3, dtype=2, bias_dtype=0, y_dtype=2, act=0, gated=0)
    assert set(kw) <= set(a)
    a.update(kw)
    return DENSE_ARGS.pack(*(a[f] for f in FIELDS))


BAD = [
    (dict(dtype=0), "dtype"), (dict(dtype=3), "dtype"), (dict(y_dtype=3), "y_dtype"), (dict(y_dtype=-1), "y_dtype"),
    (dict(bias=P, bias_dtype=5), "bias_dtype"), (dict(act=5), "act"), (dict(act=-1), "act"), (dict(M=-1), "M="),
    (dict(M=(1 << 20) + 1), "M="), (dict(K=0), "K="), (dict(K=(1 << 20) + 1, ldx=1 << 21), "K="), (dict(N=0), "N="),
    (dict(N=(1 << 20) + 1, ldy=1 << 21), "N="), (dict(ldx=63), "stride"), (dict(ldy=31), "stride"),
    (dict(residual=P, ldr=31), "stride"), (dict(x=0), "null"), (dict(w=0), "null"), (dict(y=0), "null"),
    (dict(x=P + 1), "aligned"), (dict(w=P + 1), "aligned"), (dict(y=P + 1), "aligned"), (dict(y=P + 2, y_dtype=0), "aligned"),
    (dict(residual=P + 1), "aligned"), (dict(bias=P + 2), "aligned"),
]


@pytest.mark.parametrize("kw,word", BAD)
def test_dense_linear(lib, kw, word):
    from ccut._lib import CCQ_EINVAL, last_error

    for fn in (lib.ccq_dense_linear, lib.ccq_dense_linear_grouped):
        assert fn(_args(**kw)) == CCQ_EINVAL and word in last_error()
    assert lib.ccq_dense_linear_workspace_size(_args(**kw)) == 0


@pytest.mark.parametrize("kw,word", [(dict(num_experts=0), "num_experts"), (dict(num_experts=1025), "num_experts"),
                                     (dict(offsets=0), "null"), (dict(offsets=P + 2), "aligned")])
def test_dense_linear_grouped(lib, kw, word):
    from ccut._lib import CCQ_EINVAL, last_error

    assert lib.ccq_dense_linear_grouped(_args(**kw)) == CCQ_EINVAL and word in last_error()


def test_dense_workspace(lib):
    from ccut._lib import CCQ_EINVAL, last_error

    big = dict(M=100, K=8192, N=64, ldx=8192, ldy=64)
    need = lib.ccq_dense_linear_workspace_size(_args(**big))
    assert need >= 2 * 100 * 64 * 4
    for kw in (dict(), dict(workspace=P, workspace_bytes=need - 1), dict(workspace=P + 8, workspace_bytes=need)):
        assert lib.ccq_dense_linear(_args(**big, **kw)) == CCQ_EINVAL and "workspace" in last_error()
    odd = dict(M=4000, K=515, N=700, ldx=515, ldy=700, num_experts=2)
    for size, run in ((lib.ccq_dense_linear_workspace_size, lib.ccq_dense_linear),
                      (lib.ccq_dense_linear_grouped_workspace_size, lib.ccq_dense_linear_grouped)):
        need = size(_args(**odd))
        assert need >= 4000 * 520 * 2
        assert run(_args(**odd, workspace=P, workspace_bytes=need - 1)) == CCQ_EINVAL and "workspace" in last_error()
    for M, K, N, E in ((1, 8, 1, 3), (5000, 64, 32, 3), (5000, 4096, 512, 1), (1 << 20, 8, 8, 1024)):  # aligned groups
        assert lib.ccq_dense_linear_grouped_workspace_size(_args(M=M, K=K, N=N, ldx=K, ldy=N, num_experts=E)) == 0
    for M in range(1, 17):  # what the Python entry point counts on
        for K, N in ((64, 32), (14336, 16), (1 << 20, 1), (1405, 1407)):
            assert lib.ccq_dense_linear_workspace_size(_args(M=M, K=K, N=N, ldx=K, ldy=N)) == 0
    assert lib.ccq_dense_linear(None) == CCQ_EINVAL and lib.ccq_dense_linear_grouped(None) == CCQ_EINVAL
    assert lib.ccq_dense_linear_workspace_size(None) == 0


PERMUTE_FIELDS = ("x", "ids", "rows", "position", "offsets", "weights", "y", "d_weights", "workspace", "stream",
                  "workspace_bytes", "ldx", "ldr", "T", "k", "H", "num_experts", "dtype", "y_dtype")


def _permute(**kw):
    from ccut._lib import PERMUTE_ARGS

    a = dict(x=P, ids=P, rows=P, position=P, offsets=P, weights=P, y=P, d_weights=P, workspace=0, stream=0,
             workspace_bytes=0, ldx=16, ldr=16, T=4, k=2, H=16, num_experts=3, dtype=2, y_dtype=2)
    assert set(kw) <= set(a)
    a.update(kw)
    return PERMUTE_ARGS.pack(*(a[f] for f in PERMUTE_FIELDS))


def test_empty_calls(lib):
    assert lib.ccq_dense_linear(_args(M=0)) == 0 and lib.ccq_dense_linear_grouped(_args(M=0)) == 0
    assert lib.ccq_moe_unpermute(_permute(T=0, y=0)) == 0 and lib.ccq_moe_unpermute_grad(_permute(T=0, y=0)) == 0


SIZES = [(dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(k=0), "k="), (dict(k=65), "k="), (dict(T=-1), "T="),
         (dict(T=1 << 20), "T="), (dict(T=1 << 60), "T="), (dict(H=0), "H="),
         (dict(H=(1 << 20) + 1, ldx=1 << 21, ldr=1 << 21), "H=")]


@pytest.mark.parametrize("kw,word", SIZES)
def test_permute_sizes(lib, kw, word):
    from ccut._lib import CCQ_EINVAL, last_error

    for fn in (lib.ccq_moe_permute, lib.ccq_moe_unpermute, lib.ccq_moe_unpermute_grad):
        assert fn(_permute(**kw)) == CCQ_EINVAL and word in last_error()
        assert fn(None) == CCQ_EINVAL


@pytest.mark.parametrize("kw,word", [
    (dict(num_experts=0), "num_experts"), (dict(num_experts=1025), "num_experts"), (dict(ldx=15), "stride"),
    (dict(x=0), "null"), (dict(ids=0), "null"), (dict(rows=0), "null"), (dict(position=0), "null"), (dict(offsets=0), "null"),
    (dict(T=0, offsets=0), "null"), (dict(x=P + 1), "aligned"), (dict(dtype=0, rows=P + 2), "aligned"),
    (dict(ids=P + 4), "aligned"), (dict(position=P + 2), "aligned"), (dict(offsets=P + 2), "aligned"),
    (dict(T=1 << 15), "workspace"), (dict(T=1 << 15, workspace=P, workspace_bytes=16), "workspace"),
    (dict(T=1 << 15, workspace=P + 8, workspace_bytes=1 << 30), "workspace"),
])
def test_permute(lib, kw, word):
    from ccut._lib import CCQ_EINVAL, last_error

    assert lib.ccq_moe_permute(_permute(**kw)) == CCQ_EINVAL and word in last_error()


def test_permute_workspace(lib):
    """What the Python entry point counts on."""
    for T, k in ((1, 1), (32, 64), (2048, 1), (256, 8), (292, 7)):
        assert lib.ccq_moe_permute_workspace_size(T, k, 1024) == 0
    for T, k in ((2049, 1), (1 << 20, 1), (1 << 14, 64), (293, 7)):
        assert lib.ccq_moe_permute_workspace_size(T, k, 1) > 0


@pytest.mark.parametrize("kw,word", [
    (dict(y_dtype=3), "y_dtype"), (dict(ldr=15), "stride"), (dict(rows=0), "null"), (dict(position=0), "null"),
    (dict(y=0), "null"), (dict(rows=P + 1), "aligned"), (dict(position=P + 2), "aligned"), (dict(weights=P + 2), "aligned"),
    (dict(y=P + 1), "aligned"),
])
def test_unpermute(lib, kw, word):
    from ccut._lib import CCQ_EINVAL, last_error

    assert lib.ccq_moe_unpermute(_permute(**kw)) == CCQ_EINVAL and word in last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(ldr=15), "stride"), (dict(ldx=15), "stride"), (dict(x=0), "null"), (dict(rows=0), "null"), (dict(weights=0), "null"),
    (dict(y=0), "null"), (dict(d_weights=0), "null"), (dict(position=0), "null"), (dict(x=P + 1), "aligned"),
    (dict(y=P + 1), "aligned"), (dict(d_weights=P + 2), "aligned"),
])
def test_unpermute_grad(lib, kw, word):
    from ccut._lib import CCQ_EINVAL, last_error

    assert lib.ccq_moe_unpermute_grad(_permute(**kw)) == CCQ_EINVAL and word in last_error()


def test_host_tensors_are_refused(lib):
    from ccut.blocks import moe
    from ccut.quant import dense

    x, w = torch.zeros((2, 16), dtype=torch.bfloat16), torch.zeros((8, 16), dtype=torch.bfloat16)
    plan = moe.Permutation(torch.zeros((2, 1), dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    for call in (lambda: dense.linear(x, w), lambda: dense.linear_grouped(x, plan.offsets, w[None]),
                 lambda: moe.moe_permute(x, torch.zeros((2, 1), dtype=torch.int64), 3), lambda: moe.moe_unpermute(x, plan),
                 lambda: moe.moe_permute_backward(x, plan),
                 lambda: moe.moe_unpermute_backward(x, x, plan, torch.zeros((2, 1)))):
        with pytest.raises(ValueError, match="cuda"):
            call()


def test_oracle_gradients_against_differences():
    from oracle import permute as op

    g = torch.Generator().manual_seed(0)
    ids = torch.tensor([[0, 2], [2, 2], [-1, 1], [5, -3]])
    position, offsets = op.plan(ids, 3)
    assert offsets.tolist() == [0, 1, 2, 5] and position.tolist() == [[0, 2], [3, 4], [-6, 1], [-7, -8]]
    rows, w, dy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((8, 5), (4, 2), (4, 5)))
    d_rows, d_w, _ = op.unpermute_backward(dy, rows, position, w)
    f = lambda r, v: (op.unpermute(r, position, v)[0] * dy).sum()  # noqa: E731
    for grad, arg, other in ((d_rows, rows, lambda a: f(a, w)), (d_w, w, lambda a: f(rows, a))):
        for i in range(arg.numel()):
            step = torch.zeros_like(arg)
            step.view(-1)[i] = 1e-3
            assert abs((other(arg + step) - other(arg - step)) / 2e-3 - grad.view(-1)[i]) < 1e-9


def test_oracle_activations():
    """The 64-bit activations against torch's own in 64 bits."""
    import torch.nn.functional as F

    from oracle import dense as od

    z = torch.linspace(-12, 12, 1001, dtype=torch.float64)
    for name, fn in (("relu", F.relu), ("silu", F.silu), ("gelu", F.gelu), ("gelu_tanh", lambda v: F.gelu(v, approximate="tanh"))):
        y, _, slope = od.act(z, name)
        assert torch.allclose(y, fn(z), rtol=1e-9, atol=1e-15)
        assert ((y[1:] - y[:-1]).abs() <= slope * (z[1] - z[0]) * 1.0001).all()
