"""The layer of 16-bit experts and its container on the host: what reaches the
kernels' entry points, and what is refused before (runs without a GPU)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class _Rows:
    """Rows on a device that this machine does not have."""

    dtype, shape = BF, (4, 8)

    def __init__(self, index):
        self.index = index

    def dim(self):
        return 2

    def get_device(self):
        return self.index


@pytest.mark.parametrize("forward", [False, True])
@pytest.mark.parametrize("current", [0, 1])
def test_layer_works_on_its_rows_device(monkeypatch, current, forward):
    """Routing and weights that are converted on the way go to the rows' device, whichever is current."""
    from ccut.blocks import moe

    state, seen = [current], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, state[0] = state[0], self.index

        def __exit__(self, *exc):
            state[0] = self.before

    def on_current(name, result):
        def step(*args, **kw):
            seen.append((name, state[0]))
            return result

        return step

    plan = SimpleNamespace(offsets=None)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(moe, "is_current", lambda index: index == state[0])
    monkeypatch.setattr(moe._dev, "to_device", on_current("to_device", None))
    monkeypatch.setattr(moe, "topk_softmax", on_current("topk", (None, None)))
    monkeypatch.setattr(moe, "moe_permute", on_current("permute", (None, plan)))
    monkeypatch.setattr(moe.dense, "linear_grouped", on_current("linear", None))
    monkeypatch.setattr(moe, "moe_unpermute", on_current("unpermute", "y"))
    ex = moe.DenseExperts(torch.zeros((3, 12, 8), dtype=BF), torch.zeros((3, 8, 6), dtype=BF))
    if forward:
        assert moe.moe_forward_dense(_Rows(1), None, ex, 2) == "y"
    else:
        assert moe.moe_ffn_dense(_Rows(1), None, None, ex) == "y"
    assert [name for name, _ in seen] == ["topk"] * forward + ["to_device", "permute", "linear", "linear", "to_device",
                                                               "unpermute"]
    assert all(index == 1 for _, index in seen) and state[0] == current


def test_strided_weights_are_made_dense_once():
    """Experts stored [E, in, out] come as transposed views: the container holds dense rows, so that no call copies
    them; dense ones are kept as they are."""
    from ccut.blocks import moe

    g = torch.Generator().manual_seed(0)
    gu, d = torch.randn((3, 8, 12), generator=g).to(BF), torch.randn((3, 6, 8), generator=g).to(BF)
    bgu, bd = torch.randn((12, 3), generator=g), torch.randn((3, 16), generator=g)[:, ::2]
    ex = moe.DenseExperts(gu.transpose(1, 2), d.transpose(1, 2), bgu.t(), bd)
    for t, ref in ((ex.w_gate_up, gu.transpose(1, 2)), (ex.w_down, d.transpose(1, 2)), (ex.b_gate_up, bgu.t()),
                   (ex.b_down, bd)):
        assert t.is_contiguous() and torch.equal(t, ref)
    again = moe.DenseExperts(ex.w_gate_up, ex.w_down, ex.b_gate_up, ex.b_down)
    assert again.w_gate_up is ex.w_gate_up and again.w_down is ex.w_down
    assert again.b_gate_up is ex.b_gate_up and again.b_down is ex.b_down
    assert moe.DenseExperts(ex.w_gate_up, ex.w_down).b_down is None


@pytest.mark.parametrize("shared", [None, "rows"])
@pytest.mark.parametrize("out_dtype", [torch.int32, torch.float64, torch.bool])
def test_layer_refuses_other_types_of_y(monkeypatch, out_dtype, shared):
    """With and without the shared expert's rows, before anything is computed."""
    from ccut.blocks import moe

    x = _Rows(0)
    monkeypatch.setattr(moe, "is_current", lambda index: True)
    plan = SimpleNamespace(offsets=None)
    monkeypatch.setattr(moe._dev, "to_device", lambda *args: None)
    monkeypatch.setattr(moe, "moe_permute", lambda *args: (None, plan))
    monkeypatch.setattr(moe.dense, "linear_grouped", lambda *args, **kw: None)
    monkeypatch.setattr(moe, "moe_unpermute", lambda rows, plan, weights, dtype: torch.zeros((4, 8), dtype=dtype))
    monkeypatch.setattr(moe, "_shared_rows", lambda *args: None)
    monkeypatch.setattr(moe, "shared_expert_add", lambda *args: None)
    ex = moe.DenseExperts(torch.zeros((3, 12, 8), dtype=BF), torch.zeros((3, 8, 6), dtype=BF))
    with pytest.raises(ValueError, match="y must be"):
        moe.moe_ffn_dense(x, None, None, ex, out_dtype, shared=shared)
    for ok in (None, F32, F16, BF):
        assert moe.moe_ffn_dense(x, None, None, ex, ok, shared="rows").dtype == (ok or BF)


@pytest.mark.parametrize("grouped,size", [
    (True, dict(M=16384, K=8, N=1 << 20, ldx=8, num_experts=1024)), (True, dict(M=25600, K=9, N=1 << 20, ldx=9, num_experts=128)),
    (False, dict(M=1 << 20, K=8, N=1 << 20, ldx=8)), (False, dict(M=1 << 20, K=9, N=1 << 20, ldx=9)),
])
def test_products_of_too_many_tiles_are_refused_before_any_launch(built_lib, grouped, size):
    """Also those whose rows would be copied to aligned ones first."""
    from ccut._lib import CCQ_EINVAL, DENSE_ARGS, last_error, lib

    a = dict(ldy=1 << 20, num_experts=0, ldr=0) | size
    tail = (a["ldx"], a["ldr"], a["ldy"], a["M"], a["K"], a["N"], a["num_experts"], 2, 0, 2, 0, 0)
    args = DENSE_ARGS.pack(256, 256, 0, 0, 256, 256, 256, 0, 1 << 50, *tail)
    run = lib().ccq_dense_linear_grouped if grouped else lib().ccq_dense_linear
    assert run(args) == CCQ_EINVAL and "2^22 tiles" in last_error()
    assert lib().ccq_dense_linear_kernel(args, grouped, None, None, None, None) == -1
