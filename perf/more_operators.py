"""Experts and projections held in 16 bits, as measurable cases.

``linear``     ``quant.dense.linear``: ``act(x w^T + bias)``, gated or not, ``+ residual``, of float16 or bfloat16
               rows and weights: the projections, shared experts and routers that a checkpoint leaves unquantized.
``grouped``    ``quant.dense.linear_grouped``: the same product for rows sorted by expert, each group of rows with
               its expert's weights.
``permute``    ``blocks.moe.moe_permute``: tokens sorted by expert (``back`` false), and the gradient of the tokens
               from that of the sorted rows (``back`` true).
``unpermute``  ``blocks.moe.moe_unpermute``: sorted rows back to their tokens, added under the routing weights, and
               (``back`` true) the gradients of the sorted rows and of the weights."""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "costcut-infer_amd")
_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # single-stream decode of a small model: one row through a projection
        dict(name="linear decode 1", kind="linear", M=1, K=2048, N=5632, act="none", gated=False, bias=False,
             residual=False, dtype="bf16"),
        # batched decode through the stacked gate and up projections of an 8B model's MLP
        dict(name="linear gated batch 16", kind="linear", M=16, K=4096, N=14336, act="silu", gated=True, bias=False,
             residual=False, dtype="bf16"),
        # a short prompt, every size odd, with all of the epilogue
        dict(name="linear odd 93", kind="linear", M=93, K=1405, N=1407, act="gelu", gated=False, bias=True,
             residual=True, dtype="f16"),
        # a prompt through an MLP's first projection
        dict(name="linear prefill 2048", kind="linear", M=2048, K=4096, N=14336, act="gelu_tanh", gated=False, bias=True,
             residual=False, dtype="f16"),
        # several prompts through a down projection, onto the residual stream
        dict(name="linear down 4096", kind="linear", M=4096, K=14336, N=4096, act="none", gated=False, bias=False,
             residual=True, dtype="bf16"),
        # one token through its eight experts of 128
        dict(name="grouped decode 1", kind="grouped", T=1, k=8, E=128, K=2048, N=768, act="silu", gated=True, bias=False,
             skew=0.0, bare=0, dtype="bf16"),
        # a decode batch: a few rows for each of 64 experts, some experts timed out
        dict(name="grouped batch 64", kind="grouped", T=64, k=6, E=64, K=1408, N=2048, act="none", gated=False,
             bias=True, skew=0.0, bare=9, dtype="f16"),
        # a long prompt over 128 experts, some of them far more popular than others
        dict(name="grouped prefill 4096", kind="grouped", T=4096, k=8, E=128, K=2048, N=768, act="silu", gated=True,
             bias=False, skew=2.0, bare=0, dtype="bf16"),
        # a decode batch's tokens to their experts
        dict(name="permute decode 16", kind="permute", back=False, T=16, k=6, E=64, H=2048, skew=0.0, bare=0,
             dtype="bf16"),
        # the tokens' gradient of a fine-tuning step on long sequences
        dict(name="permute gradient 4096", kind="permute", back=True, T=4096, k=8, E=128, H=2048, skew=2.0, bare=0,
             dtype="bf16"),
        # a prompt's rows back from the experts, in the reference's float32, odd hidden size, some experts timed out
        dict(name="unpermute odd 509", kind="unpermute", back=False, T=509, k=4, E=60, H=2047, skew=1.0, bare=31,
             dtype="f32"),
        # the rows' and routing weights' gradients of the large layer
        dict(name="unpermute gradient 2048", kind="unpermute", back=True, T=2048, k=8, E=256, H=7168, skew=1.0, bare=0,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["linear", "linear", "grouped", "grouped", "permute", "unpermute"])
    odd = rng.random() < 0.2
    act = rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu"])
    gated = act != "none" and rng.random() < 0.5
    dtype = rng.choice(["bf16", "f16"])
    while True:
        if kind == "linear":
            K, N = (_log(rng, 256, 14336) for _ in range(2))
            if not odd:
                K, N = (K + 15) // 16 * 16, (N + 15) // 16 * 16
            case = dict(kind=kind, M=_log(rng, 1, 8192), K=K, N=N, act=act, gated=gated, bias=rng.random() < 0.5,
                        residual=rng.random() < 0.4, dtype=dtype)
            w = work(case)
            if w["bytes"] <= 240e6 and w["flops"] <= 480e9:
                return case
            continue
        T, E = _log(rng, 1, 8192), _log(rng, 4, 256)
        k = rng.randint(1, min(8, E))
        part = dict(T=T, k=k, E=E, skew=rng.choice([0.0, 1.0, 2.0]), bare=rng.choice([0, 0, T * k // 16]), dtype=dtype)
        if kind == "grouped":
            K, N = (_log(rng, 256, 7168) for _ in range(2))
            if not odd:
                K, N = (K + 15) // 16 * 16, (N + 15) // 16 * 16
            case = dict(kind=kind, K=K, N=N, act=act, gated=gated, bias=rng.random() < 0.5, **part)
            if E * N * (1 + gated) * K <= 128 * 1536 * 2048 and 2 * T * k * N * (1 + gated) * K <= 206e9 and (
                    T * k * (K + N) <= 4096 * 8 * 2816):
                return case
            continue
        H = _log(rng, 256, 7168)
        part["dtype"] = rng.choice(["bf16", "f16", "f32"])
        case = dict(kind=kind, back=rng.random() < 0.5, H=H if odd else (H + 15) // 16 * 16, **part)
        if work(case)["bytes"] <= 500e6:
            return case


def _routing(case, seed):
    """Experts of each token (int64 [T, k], -1 for the ``bare`` ones that were left out) and what sorting by expert
    gives: the row of each assignment (the left-out ones, as ``~row``, behind the rest) and each expert's first row."""
    r = np.random.default_rng(int(seed))
    T, k, E = case["T"], case["k"], case["E"]
    logits = r.standard_normal((T, E)) + case["skew"] * r.standard_normal(E)
    ids = np.argsort(-logits, axis=1)[:, :k].astype(np.int64)
    flat = ids.reshape(-1)
    flat[r.choice(T * k, case["bare"], replace=False)] = -1
    key = np.where(flat < 0, E, flat)
    position = np.empty(T * k, np.int64)
    position[np.argsort(key, kind="stable")] = np.arange(T * k)
    position[flat < 0] = ~position[flat < 0]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])])
    return ids, position.reshape(T, k).astype(np.int32), offsets.astype(np.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)

    dt, kind = _DT[case["dtype"]], case["kind"]
    s = dict(case=case)
    if kind != "linear":
        ids, position, offsets = _routing(case, seed)
        s.update(ids=torch.from_numpy(ids).cuda(), position=torch.from_numpy(position).cuda(),
                 offsets=torch.from_numpy(offsets).cuda(), first=offsets.tolist())
    if kind in ("linear", "grouped"):
        K, N = case["K"], case["N"]
        wide = N * (1 + case["gated"])
        E = () if kind == "linear" else (case["E"],)
        rows = case["M"] if kind == "linear" else case["T"] * case["k"]
        s["x"] = normal(rows, K, dtype=dt)
        s["w"] = torch.empty((*E, wide, K), dtype=dt, device="cuda")
        for w in s["w"] if E else s["w"][None]:
            w.copy_(normal(wide, K, std=K ** -0.5))
        s["bias"] = normal(*E, wide, std=0.5, dtype=dt) if case["bias"] else None
        s["residual"] = normal(rows, N, std=2.0, dtype=dt) if case.get("residual") else None
    else:
        T, k, H = (case[n] for n in ("T", "k", "H"))
        if case["back"] == (kind == "unpermute"):
            s["x"] = normal(T, H, dtype=dt)         # tokens, or the tokens' gradient
        if kind == "unpermute" or case["back"]:
            s["rows"] = normal(T * k, H, dtype=dt)  # sorted rows, or their gradient
        s["weights"] = torch.softmax(normal(T, k), -1) if kind == "unpermute" else None
    if own:
        if _PKG not in sys.path:
            sys.path.insert(0, _PKG)
        if kind in ("linear", "grouped"):
            from ccut.quant import dense

            s["dense"] = dense
        else:
            from ccut.blocks import moe

            s["moe"], s["plan"] = moe, moe.Permutation(s["position"], s["offsets"])
    return s


def _act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return z / (1 + torch.exp(-z)) if act == "silu" else z


def _product(case, x, w, bias, residual):
    z = x.float() @ w.float().t()
    if bias is not None:
        z = z + bias.float()
    if case["gated"]:
        z = _act(z[:, :case["N"]], case["act"]) * z[:, case["N"]:]
    else:
        z = _act(z, case["act"])
    if residual is not None:
        z = z + residual.float()
    return z.to(x.dtype)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "linear":
        return {"y": _product(case, s["x"], s["w"], s["bias"], s["residual"])}
    first = s["first"]
    if kind == "grouped":
        y = torch.zeros((s["x"].shape[0], case["N"]), dtype=s["x"].dtype, device="cuda")
        for e in range(case["E"]):
            b, n = first[e], first[e + 1]
            if b < n:
                bias = s["bias"][e] if s["bias"] is not None else None
                y[b:n] = _product(case, s["x"][b:n], s["w"][e], bias, None)
        return {"y": y}
    T, k, E, H = (case[n] for n in ("T", "k", "E", "H"))
    if kind == "permute" and not case["back"]:
        flat = s["ids"].view(-1)
        key = torch.where(flat < 0, E, flat)
        order = torch.sort(key, stable=True).indices
        row = torch.empty_like(order)
        row[order] = torch.arange(T * k, device="cuda")
        rows = torch.where((flat[order] < 0)[:, None], 0, s["x"][order // k])
        offsets = (key[:, None] < torch.arange(E + 1, device="cuda")).sum(0)
        return {"rows": rows, "position": torch.where(flat < 0, ~row, row).view(T, k).int(), "offsets": offsets.int()}
    at = s["position"].long()
    kept = at >= 0
    if not (kind == "unpermute" and case["back"]):
        z = torch.where(kept[..., None], s["rows"].float()[at.clamp_min(0)], 0.0)
        if s["weights"] is not None:
            z = z * s["weights"][..., None]
        return {"x": z.sum(1).to(s["rows"].dtype)}
    dy = s["x"].float()[:, None]
    d_rows = torch.empty_like(s["rows"])
    share = torch.where(kept, s["weights"], 0.0)
    d_rows[torch.where(kept, at, ~at)] = (share[..., None] * dy).to(d_rows.dtype)
    d_weights = torch.where(kept, (s["rows"].float()[at.clamp_min(0)] * dy).sum(-1), 0.0)
    return {"rows": d_rows, "weights": d_weights}


def run(state):
    if not own:
        return _plain(state)
    s, case = state, state["case"]
    kind = case["kind"]
    act = None if case.get("act", "none") == "none" else case["act"]
    if kind == "linear":
        return {"y": s["dense"].linear(s["x"], s["w"], s["bias"], act=act, gated=case["gated"], residual=s["residual"])}
    if kind == "grouped":
        return {"y": s["dense"].linear_grouped(s["x"], s["offsets"], s["w"], s["bias"], act=act, gated=case["gated"])}
    if kind == "permute":
        if case["back"]:
            return {"x": s["moe"].moe_permute_backward(s["rows"], s["plan"])}
        rows, plan = s["moe"].moe_permute(s["x"], s["ids"], case["E"])
        return {"rows": rows, "position": plan.position, "offsets": plan.offsets}
    if not case["back"]:
        return {"x": s["moe"].moe_unpermute(s["rows"], s["plan"], s["weights"])}
    d_rows, d_weights = s["moe"].moe_unpermute_backward(s["x"], s["rows"], s["plan"], s["weights"])
    return {"rows": d_rows, "weights": d_weights}


def work(case):
    e = _SIZE[case["dtype"]]
    if case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        wide = N * (1 + case["gated"])
        values = M * K + wide * K + M * N * (1 + case["residual"]) + wide * case["bias"]
        return {"bytes": values * e, "flops": 2 * M * wide * K}
    T, k, E = case["T"], case["k"], case["E"]
    rows = T * k - case["bare"]
    if case["kind"] == "grouped":
        K, N = case["K"], case["N"]
        wide = N * (1 + case["gated"])
        used = int((np.diff(_routing(case, 0)[2]) > 0).sum())
        values = rows * K + used * wide * (K + case["bias"]) + T * k * N
        return {"bytes": values * e + 4 * E, "flops": 2 * rows * wide * K}
    H = case["H"]
    if case["kind"] == "permute":
        # the experts' numbers in and the plan out, or the plan in
        small = T * k * 4 + (0 if case["back"] else T * k * 8 + E * 4)
        moved = (T + rows if case["back"] else T + T * k) * H
        return {"bytes": moved * e + small, "flops": rows * H if case["back"] else 0}
    if case["back"]:
        return {"bytes": (T + rows + T * k) * H * e + T * k * 12, "flops": 3 * rows * H}
    return {"bytes": (rows + T) * H * e + T * k * 8, "flops": 2 * rows * H}


def _exact_act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * z * (1 + 0.044715 * z ** 2))
    return z * torch.sigmoid(z) if act == "silu" else z


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("linear", "grouped"):
        N = case["N"]
        groups = [(0, case["M"], s["w"], s["bias"])] if kind == "linear" else [
            (s["first"][e], s["first"][e + 1], s["w"][e], s["bias"][e] if case["bias"] else None)
            for e in range(case["E"])]
        y = torch.zeros((s["x"].shape[0], N), dtype=torch.float64, device="cuda")
        for b, n, w, bias in groups:
            if n > b:
                x = s["x"][b:n].double()
                parts = [x.mm(p.double().t().contiguous()) for p in w.split(N)]
                if bias is not None:
                    parts = [p + q.double() for p, q in zip(parts, bias.split(N))]
                y[b:n] = _exact_act(parts[0], case["act"]) * (parts[1] if case["gated"] else 1)
        if s.get("residual") is not None:
            y += s["residual"].double()
        return {"y": y}
    T, k, E, H = (case[n] for n in ("T", "k", "E", "H"))
    if kind == "permute" and not case["back"]:
        ids, row = s["ids"].cpu(), 0
        rows = torch.zeros((T * k, H), dtype=torch.float64, device="cuda")
        position, offsets = torch.empty((T, k), dtype=torch.int32), [0]
        for e in [*range(E), -1]:
            t, slot = (ids == e).nonzero(as_tuple=True)
            n = row + len(t)
            at = torch.arange(row, n, dtype=torch.int32)
            position[t, slot] = at if e >= 0 else -1 - at
            if e >= 0:
                rows[row:n] = s["x"][t.cuda()].double()
                offsets.append(n)
            row = n
        return {"rows": rows, "position": position.cuda(), "offsets": torch.tensor(offsets, dtype=torch.int32).cuda()}
    d_rows = torch.zeros((T * k, H), dtype=torch.float64, device="cuda")
    d_weights = torch.zeros((T, k), dtype=torch.float64, device="cuda")
    x = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    for slot in range(k):
        t = (s["position"][:, slot] >= 0).nonzero().view(-1)
        at = s["position"][t, slot].long()
        share = s["weights"][t, slot].double()[:, None] if kind == "unpermute" else 1.0
        if kind == "unpermute" and case["back"]:
            dy = s["x"][t].double()
            d_rows[at] = dy * share
            d_weights[t, slot] = s["rows"][at].double().mul(dy).sum(1)
        else:
            x[t] += s["rows"][at].double() * share
    if kind == "unpermute" and case["back"]:
        return {"rows": d_rows, "weights": d_weights}
    return {"x": x}
