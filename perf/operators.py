"""The measured cases of the 4-bit expert weights and of the few-token MoE layer.

Four operators, each in a plain form (elementary torch operations) and through
the framework's entry points:

* ``quantize``: a weight matrix in groups of 4-bit codes along K, with a bf16
  scale (and, asymmetric, a zero point) for each row and group, and the values
  that the codes stand for;
* ``linear``: y = x W^T + b with W in that form;
* ``gated_mlp``: one SwiGLU expert, down(silu(gate x) * (up x)), in that form;
* ``moe``: a whole mixture-of-experts layer for a few tokens - a dense gate,
  softmax, top-k and the experts' weighted sum - or its experts alone behind
  a router that has already chosen; experts in 4-bit groups or ternary.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _package():
    """The framework's package folder on the import path (its name is no Python identifier)."""
    path = str(Path(__file__).resolve().parents[1] / "spectral-ai_b200")
    if path not in sys.path:
        sys.path.insert(0, path)


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one expert's gate matrix, quantised as a checkpoint is loaded
        {"name": "quantize expert", "op": "quantize", "N": 1024, "K": 2048, "group": 128, "zeros": False, "dtype": "bf16"},
        # a wide fp32 layer with zero points, rows that end inside a group
        {"name": "quantize wide ragged", "op": "quantize", "N": 8192, "K": 4100, "group": 64, "zeros": True, "dtype": "fp32"},
        # one token through a square projection: latency
        {"name": "linear 1 token", "op": "linear", "M": 1, "K": 2048, "N": 2048, "group": 128, "zeros": False, "bias": False, "dtype": "bf16"},
        # a small decoding batch through a large projection: weight bandwidth
        {"name": "linear 8 tokens", "op": "linear", "M": 8, "K": 4096, "N": 8192, "group": 64, "zeros": True, "bias": True, "dtype": "bf16"},
        # odd sizes, the smallest groups, fp32 activations
        {"name": "linear odd fp32", "op": "linear", "M": 5, "K": 1000, "N": 777, "group": 32, "zeros": True, "bias": True, "dtype": "fp32"},
        # a long prompt: the matrix product
        {"name": "linear prompt", "op": "linear", "M": 2048, "K": 2048, "N": 4096, "group": 128, "zeros": False, "bias": False, "dtype": "bf16"},
        # one expert, one token
        {"name": "mlp 1 token", "op": "gated_mlp", "M": 1, "H": 2048, "I": 1024, "group": 128, "zeros": False, "dtype": "bf16"},
        # one expert, a prompt's ragged share of tokens
        {"name": "mlp 300 tokens", "op": "gated_mlp", "M": 300, "H": 2048, "I": 1024, "group": 64, "zeros": True, "dtype": "bf16"},
        # decoding one sequence: gate, top-8 of 64 and the experts
        {"name": "moe 1 token", "op": "moe", "B": 1, "E": 64, "k": 8, "H": 2048, "I": 1024, "weights": "group4", "group": 128, "zeros": False, "gate": True, "norm": False, "dtype": "bf16"},
        # a decoding batch that touches nearly every expert
        {"name": "moe 64 tokens", "op": "moe", "B": 64, "E": 64, "k": 8, "H": 2048, "I": 1024, "weights": "group4", "group": 128, "zeros": True, "gate": True, "norm": True, "dtype": "bf16"},
        # ternary experts behind a router that has chosen, one token
        {"name": "moe ternary routed 1", "op": "moe", "B": 1, "E": 64, "k": 8, "H": 2048, "I": 1024, "weights": "ternary", "group": 0, "zeros": False, "gate": False, "norm": False, "dtype": "bf16"},
        # ternary experts with their gate, a batch
        {"name": "moe ternary 24 tokens", "op": "moe", "B": 24, "E": 64, "k": 8, "H": 2048, "I": 1024, "weights": "ternary", "group": 0, "zeros": False, "gate": True, "norm": False, "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi):
    """A size: mostly multiples of 64, as models have them, else any number."""
    n = _spread(rng, lo, hi)
    return n if rng.random() < 0.4 else min(hi, max(lo, (n + 32) // 64 * 64))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "gated_mlp", "moe", "moe"])
    group, zeros = rng.choice([32, 64, 128]), rng.random() < 0.5
    dtype = "fp32" if rng.random() < 0.25 else "bf16"
    if op == "quantize":
        return {"op": op, "N": _size(rng, 64, 8192), "K": _size(rng, 64, 4096), "group": group, "zeros": zeros, "dtype": dtype}
    if op == "linear":
        return {"op": op, "M": _spread(rng, 1, 2048), "K": _size(rng, 64, 2048), "N": _size(rng, 64, 4096), "group": group, "zeros": zeros, "bias": rng.random() < 0.5,
                "dtype": dtype}
    if op == "gated_mlp":
        return {"op": op, "M": _spread(rng, 1, 512), "H": _size(rng, 128, 2048), "I": _size(rng, 64, 1024), "group": group, "zeros": zeros, "dtype": dtype}
    E = rng.choice([8, 16, 40, 64])
    ternary = rng.random() < 0.5
    return {"op": op, "B": _spread(rng, 1, 64), "E": E, "k": rng.randint(1, 8), "H": _size(rng, 128, 2048), "I": _size(rng, 64, 1024), "weights": "ternary" if ternary else "group4",
            "group": 0 if ternary else group, "zeros": zeros and not ternary, "gate": rng.random() < 0.6, "norm": rng.random() < 0.5, "dtype": dtype}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _activations(g, rows, cols, dtype):
    """Hidden states: unit normal with a few channels that are much larger."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    return (x * torch.where(loud, 6.0, 1.0)).to(dtype)


def _codes(g, shape, K, group, zeros):
    """Codes, scales and zero points of a quantised normal matrix [..., K] (all shapes but the last are rows)."""
    groups = -(-K // group)
    z = torch.randint(5, 11, (*shape, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    mid = z.repeat_interleave(group, -1)[..., :K] if zeros else 8
    codes = (torch.randn(*shape, K, generator=g, device="cuda") * 2.6 + mid).round_().clamp_(0, 15).to(torch.uint8)
    scales = ((torch.rand(*shape, groups, generator=g, device="cuda") + 0.5) / (2.6 * math.sqrt(K))).bfloat16()
    return {"codes": codes, "scales": scales, "zeros": z, "group": group}


def _ternary(g, E, N, K):
    t = torch.randint(-1, 2, (E, N, K), generator=g, device="cuda", dtype=torch.int8)
    return {"t": t, "scale": (torch.rand(E, N, generator=g, device="cuda") + 0.5) / math.sqrt(K)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, op = case, case["op"]
    s = {"case": c}
    if op == "quantize":
        w = torch.randn(c["N"], c["K"], generator=g, device="cuda") / math.sqrt(c["K"])
        s["w"] = w.to(DTYPES[c["dtype"]])
        return s
    if op == "linear":
        s["x"] = _activations(g, c["M"], c["K"], DTYPES[c["dtype"]])
        s["w"] = _codes(g, (c["N"],), c["K"], c["group"], c["zeros"])
        s["bias"] = torch.randn(c["N"], generator=g, device="cuda") if c["bias"] else None
    elif op == "gated_mlp":
        s["x"] = _activations(g, c["M"], c["H"], DTYPES[c["dtype"]])
        shapes = {"gate": (c["I"], c["H"]), "up": (c["I"], c["H"]), "down": (c["H"], c["I"])}
        s |= {n: _codes(g, (rows,), cols, c["group"], c["zeros"]) for n, (rows, cols) in shapes.items()}
    else:
        s["x"] = _activations(g, c["B"], c["H"], DTYPES[c["dtype"]])
        shapes = {"gate": (c["I"], c["H"]), "up": (c["I"], c["H"]), "down": (c["H"], c["I"])}
        for n, (rows, cols) in shapes.items():
            s[n] = _ternary(g, c["E"], rows, cols) if c["weights"] == "ternary" else _codes(g, (c["E"], rows), cols, c["group"], c["zeros"])
        if c["gate"]:
            s["gate_weight"] = (torch.randn(c["E"], c["H"], generator=g, device="cuda") / math.sqrt(c["H"])).to(DTYPES[c["dtype"]])
        else:
            p = torch.randn(c["B"], c["E"], generator=g, device="cuda").softmax(-1)
            top = p.topk(c["k"], dim=-1)
            s["ids"], s["weights"] = top.indices.int(), top.values
    if own:  # the weights in the framework's layout, as a program lays them out once when it loads them
        _package()
        from sb200 import group4, moe, ternary

        def packed(m):
            return group4.Group4Matrix.pack(m["codes"], m["scales"], m["zeros"], group=m["group"])

        if op == "linear":
            s["matrix"] = packed(s["w"])
        elif op == "gated_mlp":
            s["matrices"] = [packed(s[n]) for n in ("gate", "up", "down")]
        else:
            if c["weights"] == "ternary":
                experts = ternary.TernaryExperts.from_tensors(*(s[n]["t"] for n in ("gate", "up", "down")), *(s[n]["scale"] for n in ("gate", "up", "down")))
            else:
                experts = group4.Group4Experts.pack(*({k: s[n][k] for k in ("codes", "scales", "zeros")} for n in ("gate", "up", "down")), group=c["group"])
            s["experts"] = experts
            if c["gate"]:
                s["layer"] = moe.FewTokenMoE(experts, s["gate_weight"], top_k=c["k"], norm_topk=c["norm"])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _run_own(s):
    _package()
    from sb200 import group4
    c, op = s["case"], s["case"]["op"]
    if op == "quantize":
        m, values = group4.quantize(s["w"], group=c["group"], symmetric=not c["zeros"], values=True)
        return {"values": values, "scales": m.scales, "zeros": m.zeros}
    if op == "linear":
        return group4.linear(s["x"], s["matrix"], s["bias"])
    if op == "gated_mlp":
        return group4.gated_mlp(s["x"], *s["matrices"])
    if c["gate"]:
        out, ids, weights = s["layer"](s["x"], routing=True)
        return {"out": out, "ids": ids, "weights": weights}
    return {"out": s["experts"].forward_few(s["x"], s["ids"], s["weights"], out_dtype=s["x"].dtype)}


def _quantize(w, group, zeros):
    """Groups along K of row n: scale s = absmax/7 (asymmetric: (max - min)/15, zero
    among them), rounded to fp32 and then bf16; code round(w/s) + zero, ties to even,
    in 0..15.  The quotients are taken in 64 bits: they decide a rounding."""
    N, K = w.shape
    G = -(-K // group)
    v = torch.nn.functional.pad(w.float(), (0, G * group - K)).view(N, G, group)
    if zeros:
        lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
        scales = ((hi - lo).double() / 15).float().bfloat16()
        s = scales.double()
        z = torch.where(s > 0, (-lo.double() / s).round(), 8.0).clamp(0, 15)
    else:
        scales = (v.abs().amax(-1).double() / 7).float().bfloat16()
        s = scales.double()
        z = torch.full_like(s, 8.0)
    q = torch.where(s[..., None] > 0, (v.double() / s[..., None]).round(), 0.0) + z[..., None]
    q = q.clamp(0, 15)
    values = ((q - z[..., None]).float() * scales.float()[..., None]).view(N, -1)[:, :K]
    return {"values": values.contiguous(), "scales": scales, "zeros": z.to(torch.uint8) if zeros else None}


def _values(m, at=None):
    """fp32 values of 4-bit codes or ternary weights, whole or of the experts `at`."""
    take = (lambda t: t) if at is None else (lambda t: t[at])
    if "t" in m:
        return take(m["t"]).float() * take(m["scale"])[..., None]
    codes, K, group = take(m["codes"]), m["codes"].shape[-1], m["group"]
    spread = lambda t: t.repeat_interleave(group, -1)[..., :K]  # noqa: E731
    zero = 8.0 if m["zeros"] is None else spread(take(m["zeros"])).float()
    return (codes.float() - zero) * spread(take(m["scales"]).float())


def _silu(v):
    return v / (1 + torch.exp(-v))


def _top(logits, k, norm):
    """Softmax over the experts, its k largest (the lower expert among equals), as
    they are or divided by their sum."""
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    return ids.int(), w / w.sum(-1, keepdim=True) if norm else w


def _experts(x, ids, weights, gate, up, down, E):
    """sum_j weights[t, j] * expert_{ids[t, j]}(x[t]): entry by entry where there are
    fewer entries than experts, else every expert on every token."""
    B, k = ids.shape
    if B * k <= E:
        at = ids.reshape(-1).long()
        xr = x.repeat_interleave(k, 0)[..., None]
        h = _silu(_values(gate, at) @ xr) * (_values(up, at) @ xr)
        return ((_values(down, at) @ h).view(B, k, -1) * weights[..., None]).sum(1)
    h = _silu(x @ _values(gate).mT) * (x @ _values(up).mT)
    we = torch.zeros(B, E, device=x.device).scatter_add_(1, ids.long(), weights)
    return ((h @ _values(down).mT) * we.t()[..., None]).sum(0)


def run(state):
    if own:
        return _run_own(state)
    s, c, op = state, state["case"], state["case"]["op"]
    if op == "quantize":
        return _quantize(s["w"], c["group"], c["zeros"])
    x = s["x"].float()
    if op == "linear":
        y = x @ _values(s["w"]).t()
        return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)
    if op == "gated_mlp":
        h = _silu(x @ _values(s["gate"]).t()) * (x @ _values(s["up"]).t())
        return (h @ _values(s["down"]).t()).to(s["x"].dtype)
    if not c["gate"]:
        return {"out": _experts(x, s["ids"], s["weights"], s["gate"], s["up"], s["down"], c["E"]).to(s["x"].dtype)}
    # the gate's sums in 64 bits, rounded once: they decide an order
    logits = (s["x"].double() @ s["gate_weight"].double().t()).float()
    ids, weights = _top(logits, c["k"], c["norm"])
    return {"out": _experts(x, ids, weights, s["gate"], s["up"], s["down"], c["E"]).to(s["x"].dtype), "ids": ids, "weights": weights}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _bytes4(N, K, group, zeros):
    return N * K / 2 + N * -(-K // group) * (3 if zeros else 2)


def work(case):
    c, op = case, case["op"]
    e = 2 if c["dtype"] == "bf16" else 4
    if op == "quantize":  # the matrix in, its codes' values (fp32), scales and zero points out
        return {"bytes": c["N"] * c["K"] * (e + 4) + _bytes4(c["N"], c["K"], c["group"], c["zeros"]), "flops": 3 * c["N"] * c["K"]}
    if op == "linear":
        return {"bytes": _bytes4(c["N"], c["K"], c["group"], c["zeros"]) + c["M"] * (c["K"] + c["N"]) * e + 4 * c["N"] * c["bias"], "flops": 2 * c["M"] * c["N"] * c["K"]}
    H, I = c["H"], c["I"]
    if op == "gated_mlp":
        w = 2 * _bytes4(I, H, c["group"], c["zeros"]) + _bytes4(H, I, c["group"], c["zeros"])
        return {"bytes": w + 2 * c["M"] * H * e, "flops": 6 * c["M"] * H * I}
    if c["weights"] == "ternary":
        w = 3 * H * I / 4 + 4 * (2 * I + H)
    else:
        w = 2 * _bytes4(I, H, c["group"], c["zeros"]) + _bytes4(H, I, c["group"], c["zeros"])
    k = min(c["k"], c["E"])
    touched = c["E"] * (1 - (1 - k / c["E"]) ** c["B"])  # experts that a batch of evenly spread tokens needs
    gate = c["E"] * H * e if c["gate"] else 0
    return {"bytes": touched * w + gate + 2 * c["B"] * H * e + 8 * c["B"] * k, "flops": 6 * c["B"] * k * H * I + (2 * c["B"] * c["E"] * H if c["gate"] else 0)}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------

def _exact_weights(m, e=None):
    """Values in float64: (code - zero) * scale of the element's group, or t * scale of its row."""
    pick = lambda t: None if t is None else (t if e is None else t[e])  # noqa: E731
    if "t" in m:
        return pick(m["t"]).double() * pick(m["scale"]).double().unsqueeze(-1)
    codes = pick(m["codes"]).double()
    of = torch.arange(codes.shape[-1], device=codes.device) // m["group"]
    zero = pick(m["zeros"])
    codes -= 8.0 if zero is None else zero.double()[..., of]
    return codes * pick(m["scales"]).double()[..., of]


def exact(case, seed):
    c, op, s = case, case["op"], prepare(case, seed)
    if op == "quantize":
        w = s["w"].double()
        N, K = w.shape
        of = torch.arange(K, device=w.device) // c["group"]
        G = int(of[-1]) + 1
        at = of.expand(N, K)
        start = torch.zeros(N, G, dtype=torch.float64, device=w.device)
        hi = start.scatter_reduce(1, at, w, "amax")
        lo = start.scatter_reduce(1, at, w, "amin")
        span = (hi - lo).float().double() / 15 if c["zeros"] else torch.maximum(hi, -lo) / 7
        scales = span.float().bfloat16().double()
        zero = torch.full_like(scales, 8.0)
        if c["zeros"]:
            zero = torch.where(scales == 0, zero, torch.clamp(torch.round(-lo / scales), 0, 15))
        sk, zk = scales[:, of], zero[:, of]
        code = torch.clamp(torch.where(sk == 0, zk, torch.round(w / sk) + zk), 0, 15)
        return {"values": (code - zk) * sk, "scales": scales, "zeros": None}
    x = s["x"].double()
    if op == "linear":
        y = torch.einsum("mk,nk->mn", x, _exact_weights(s["w"]))
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "gated_mlp":
        g, u = (torch.einsum("mk,nk->mn", x, _exact_weights(s[n])) for n in ("gate", "up"))
        return torch.einsum("mk,nk->mn", g * torch.sigmoid(g) * u, _exact_weights(s["down"]))
    if c["gate"]:
        logits = torch.einsum("bh,eh->be", x, s["gate_weight"].double())
        p, k = torch.softmax(logits, -1), min(c["k"], c["E"])
        top = torch.topk(p, k, dim=-1)
        ids, weights = top.indices, top.values / top.values.sum(-1, keepdim=True) if c["norm"] else top.values
    else:
        ids, weights = s["ids"].long(), s["weights"].double()
    out = torch.zeros(c["B"], c["H"], dtype=torch.float64, device=x.device)
    for e in ids.unique().tolist():
        t, j = (ids == e).nonzero(as_tuple=True)
        g, u = (torch.einsum("mk,nk->mn", x[t], _exact_weights(s[n], e)) for n in ("gate", "up"))
        y = torch.einsum("mk,nk->mn", g * torch.sigmoid(g) * u, _exact_weights(s["down"], e))
        out.index_add_(0, t, y * weights[t, j, None])
    return {"out": out, "ids": None, "weights": weights} if c["gate"] else {"out": out}
