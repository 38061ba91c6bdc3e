"""The operators beside a quantized Linear, as measurable cases: the RMS norm
that makes its 8-bit input, and the low-rank adapters added to its output.

``norm``  ``blocks.norm``: residual addition, RMS norm, and 8-bit rows with
          scales -- e4m3 with a scale per token and 128 channels (what the
          block-FP8 linears multiply) or int8 with a scale per token (what the
          W8A8 linear multiplies) -- with the normalized rows in the input's
          type beside them where adapters or a router read those.
``lora``  ``quant.lora``: ``y[t] += scale * B (A x[t])`` with the adapter of
          each token, in place on a projection's output."""

from __future__ import annotations

import random
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "costcut-infer_amd")
_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-6


def listed():
    return [
        # single-stream decode of a small model: the smallest call, bound by latency
        dict(name="norm fp8 decode 1", kind="norm", fmt="fp8", T=1, H=2048, dtype="bf16", residual=True, normed=False),
        # a serving batch in front of a W8A8 projection
        dict(name="norm int8 batch 37", kind="norm", fmt="int8", T=37, H=4096, dtype="f16", residual=True,
             normed=False),
        # float32 rows (what the reference's callers hand over) in front of a block-FP8 MoE layer
        dict(name="norm fp8 f32 93", kind="norm", fmt="fp8", T=93, H=7168, dtype="f32", residual=False, normed=True),
        # a prompt of odd length and a hidden size that no vector divides
        dict(name="norm int8 odd 1021", kind="norm", fmt="int8", T=1021, H=2047, dtype="bf16", residual=True,
             normed=True),
        # prompt processing of the large block-FP8 layer, with adapters beside it
        dict(name="norm fp8 prefill 4096", kind="norm", fmt="fp8", T=4096, H=7168, dtype="bf16", residual=True,
             normed=True),
        # one request with one adapter
        dict(name="lora decode 1", kind="lora", T=1, K=2048, N=5632, R=16, L=4, runs=0, bare=0, dtype="f16",
             weights="f16", ranks=False),
        # batched decode, an adapter per request, on the MLP projection of an 8B model
        dict(name="lora decode 16", kind="lora", T=16, K=4096, N=14336, R=16, L=16, runs=0, bare=0, dtype="bf16",
             weights="bf16", ranks=False),
        # a larger batch: adapters of several ranks, shared by some requests, and requests without one
        dict(name="lora batch 93 ranks", kind="lora", T=93, K=4096, N=4096, R=64, L=32, runs=0, bare=13, dtype="bf16",
             weights="bf16", ranks=True),
        # float32 rows of LinearProj, nothing aligned
        dict(name="lora f32 odd 41", kind="lora", T=41, K=1405, N=1407, R=12, L=5, runs=0, bare=3, dtype="f32",
             weights="bf16", ranks=False),
        # a big decode batch over few adapters of low rank
        dict(name="lora batch 512", kind="lora", T=512, K=2048, N=1408, R=8, L=8, runs=0, bare=64, dtype="f16",
             weights="f16", ranks=False),
        # prompts of five requests, one behind the other
        dict(name="lora prefill 2048", kind="lora", T=2048, K=4096, N=14336, R=16, L=8, runs=5, bare=0, dtype="bf16",
             weights="bf16", ranks=False),
        # long prompts and a high rank on a down projection
        dict(name="lora prefill 4096 r128", kind="lora", T=4096, K=14336, N=4096, R=128, L=4, runs=3, bare=200,
             dtype="bf16", weights="bf16", ranks=False),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    if rng.random() < 0.45:
        fmt = rng.choice(["fp8", "int8"])
        dtype = rng.choice(["bf16", "f16", "f32"])
        H = 128 * _log(rng, 2, 64) if fmt == "fp8" else _log(rng, 64, 8192)
        most = 4096 * 7168 * 2 // _SIZE[dtype]
        T = _log(rng, 1, min(8192, most // H))
        return dict(kind="norm", fmt=fmt, T=T, H=H, dtype=dtype, residual=rng.random() < 0.7,
                    normed=rng.random() < 0.4)
    while True:
        odd = rng.random() < 0.2
        K, N = (_log(rng, 256, 14336) for _ in range(2))
        if not odd:
            K, N = (K + 15) // 16 * 16, (N + 15) // 16 * 16
        R = rng.randint(1, 48) if odd else rng.choice([8, 16, 16, 32, 64, 128])
        L = _log(rng, 1, 64)
        T = _log(rng, 1, 4096)
        dtype, weights = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
        runs = rng.randint(1, 8) if T >= 64 and rng.random() < 0.6 else 0
        case = dict(kind="lora", T=T, K=K, N=N, R=R, L=L, runs=runs, bare=rng.choice([0, T // 8]), dtype=dtype,
                    weights=weights, ranks=rng.random() < 0.3)
        if work(case)["bytes"] <= 200e6 and T * L * R * (K + N) <= 4e11:
            return case


def _index(case, seed):
    """The adapter of each token: ``runs`` prompts of uneven lengths one behind the other, or (0) tokens of all
    adapters in mixed order; ``bare`` of the tokens have none."""
    r = random.Random(seed)
    T, L = case["T"], case["L"]
    if case["runs"]:
        cuts = sorted(r.sample(range(1, T), min(case["runs"], T) - 1))
        ends = cuts + [T]
        first = r.randrange(L)
        index = [(first + i) % L for i, (b, e) in enumerate(zip([0] + cuts, ends)) for _ in range(e - b)]
        at = r.randrange(T - case["bare"] + 1)
        index[at:at + case["bare"]] = [-1] * case["bare"]
    else:
        index = [i % L for i in range(T - case["bare"])] + [-1] * case["bare"]
        r.shuffle(index)
    return index


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    dt = _DT[case["dtype"]]
    if case["kind"] == "norm":
        T, H = case["T"], case["H"]
        x = normal(T, H, dtype=dt)
        # a residual stream: some channels far larger than the others
        channel = torch.exp(normal(H, std=0.7))
        residual = (normal(T, H) * channel).to(dt) if case["residual"] else None
        state = dict(case=case, x=x, residual=residual, weight=(1 + normal(H, std=0.1)).to(dt))
    else:
        T, K, N, R, L = (case[k] for k in ("T", "K", "N", "R", "L"))
        wt = _DT[case["weights"]]
        r = random.Random(seed)
        rank = torch.tensor([r.randint(max(1, R // 4), R) for _ in range(L)], dtype=torch.int32).cuda()
        state = dict(case=case, x=normal(T, K, dtype=dt), y=normal(T, N, dtype=dt),
                     a=normal(L, R, K, std=K ** -0.5, dtype=wt), b=normal(L, N, R, std=0.05, dtype=wt),
                     scale=torch.tensor([r.choice([0.5, 1.0, 2.0]) for _ in range(L)]).cuda(),
                     rank=rank if case["ranks"] else None,
                     index=torch.tensor(_index(case, seed), dtype=torch.int64).cuda())
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        from ccut.blocks import norm
        from ccut.quant import lora

        state["norm"], state["lora"] = norm, lora
        if case["kind"] == "lora":  # the handle that a program keeps: it refers to the same tensors
            state["adapters"] = lora.LoraAdapters(state["a"], state["b"], state["scale"], state["rank"])
    return state


def _norm_plain(s):
    case = s["case"]
    T, H = case["T"], case["H"]
    x, w = s["x"].float(), s["weight"].float()
    out = {}
    if case["residual"]:
        x = x + s["residual"].float()
        out["residual"] = x.to(s["x"].dtype)
    rstd = (x.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    p = x * w
    if case["normed"]:
        out["y"] = (p * rstd).to(s["x"].dtype)
    if case["fmt"] == "fp8":
        p = p.view(T, H // 128, 128)
        m = p.abs().amax(-1, keepdim=True).clamp_min(1e-30)
        out["q"] = (p * (torch.full_like(m, 448.0) / m)).to(torch.float8_e4m3fn).view(T, H)
        out["scale"] = (m * rstd.unsqueeze(-1) / 448.0).view(T, H // 128)
    else:
        # the codes are whole numbers: they go by the products alone, which are rounded once
        m = p.abs().amax(-1, keepdim=True).clamp_min(1e-30)
        out["q"] = (p * (torch.full_like(m, 127.0) / m)).round().clamp(-127, 127).to(torch.int8)
        out["scale"] = (m * rstd / 127.0).view(T)
    return out


def _lora_plain(s):
    x, a, b, index = s["x"].float(), s["a"].float(), s["b"].float(), s["index"]
    L, R, K = a.shape
    p = (x @ a.view(L * R, K).t()).view(-1, L, R)
    taken = (index[:, None] == torch.arange(L, device="cuda"))[:, :, None]
    if s["rank"] is not None:
        taken = taken & (torch.arange(R, device="cuda") < s["rank"][:, None])
    p = torch.where(taken, p * s["scale"][:, None], 0.0)
    delta = p.view(-1, L * R) @ b.permute(0, 2, 1).reshape(L * R, -1)
    s["y"].copy_(s["y"].float() + delta)
    return {"y": s["y"]}


def run(state):
    case = state["case"]
    if not own:
        return _norm_plain(state) if case["kind"] == "norm" else _lora_plain(state)
    if case["kind"] == "lora":
        return {"y": state["lora"].add_(state["y"], state["x"], state["adapters"], state["index"])}
    rows = state["norm"].rms_norm_fp8 if case["fmt"] == "fp8" else state["norm"].rms_norm_int8
    q, scale, y, residual = rows(state["x"], state["weight"], _EPS, residual=state["residual"],
                                 normed=case["normed"])
    out = {"q": q.view(torch.float8_e4m3fn) if case["fmt"] == "fp8" else q, "scale": scale}
    if case["normed"]:
        out["y"] = y
    if case["residual"]:
        out["residual"] = residual
    return out


def work(case):
    e = _SIZE[case["dtype"]]
    if case["kind"] == "norm":
        T, H = case["T"], case["H"]
        scales = T * (H // 128 if case["fmt"] == "fp8" else 1) * 4
        rows = e * (1 + 2 * case["residual"] + case["normed"]) + 1
        return {"bytes": T * H * rows + scales + H * e, "flops": 8 * T * H}
    T, K, N, R, L = (case[k] for k in ("T", "K", "N", "R", "L"))
    rows = T - case["bare"]
    used = min(L, rows if not case["runs"] else case["runs"])
    return {"bytes": rows * (K + 2 * N) * e + T * 8 + used * R * (K + N) * 2, "flops": 2 * rows * R * (K + N)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "lora":
        x, y = s["x"].double(), s["y"].double()
        for i in s["index"].unique().tolist():
            if i >= 0:
                at = (s["index"] == i).nonzero().view(-1)
                r = int(s["rank"][i]) if s["rank"] is not None else case["R"]
                inner = x[at] @ s["a"][i, :r].double().t()
                y[at] += float(s["scale"][i]) * (inner @ s["b"][i, :, :r].double().t())
        return {"y": y}
    x = s["x"].double()
    out = {}
    if s["residual"] is not None:
        x += s["residual"].double()
        out["residual"] = x.clone()
    norm = x.mul(x).sum(-1, keepdim=True).div(case["H"]).add(_EPS).sqrt()
    y = x / norm * s["weight"].double()
    if case["normed"]:
        out["y"] = y
    if case["fmt"] == "fp8":
        groups = y.view(case["T"], -1, 128)
        scale = groups.abs().amax(-1) / 448
        out["q"] = (groups / scale[..., None]).to(torch.float8_e4m3fn).double().view(y.shape)
    else:
        scale = y.abs().amax(-1) / 127
        out["q"] = (y / scale[:, None]).round().to(torch.int8)
    out["scale"] = scale
    return out
