"""Weights in 4-bit groups and the few-token MoE layer, restated in float64 numpy.

Beside each product stands a bound of what fp32 sums and the stated roundings may
move it by, from the same inputs, so that a test's tolerance is derived and not
chosen: an m16n8k16 step adds 16 exact products to an fp32 sum and rounds towards
zero, so after n steps (and the additions that join partial sums) a sum is within
n * 2^-23 of the sum of its terms' magnitudes.
"""

from __future__ import annotations

import numpy as np

U = {"bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}  # half a step of each output type
STEP = 2.0 ** -23


def bf16(v):
    """Round fp32 values to bf16 (nearest, ties to even), as float64."""
    b = np.asarray(v, np.float32).view(np.uint32).astype(np.uint64)
    b = (b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000
    return b.astype(np.uint32).view(np.float32).astype(np.float64)


def quantize(w, group, symmetric=True):
    """(codes uint8 [N,K], scales float64 of bf16 values [N,G], zeros uint8 [N,G])."""
    w = np.asarray(w, np.float64)
    N, K = w.shape
    G = -(-K // group)
    codes, scales, zeros = np.zeros((N, K), np.uint8), np.zeros((N, G)), np.full((N, G), 8, np.uint8)
    for g in range(G):
        v = w[:, g * group:(g + 1) * group]
        if symmetric:
            s = bf16((np.abs(v).max(1) / 7).astype(np.float32))
        else:
            lo, hi = np.minimum(v.min(1), 0), np.maximum(v.max(1), 0)
            s = bf16(((hi - lo).astype(np.float32).astype(np.float64) / 15).astype(np.float32))
        safe = np.where(s > 0, s, 1.0)
        if not symmetric:
            zeros[:, g] = np.where(s > 0, np.clip(np.rint(-lo / safe), 0, 15), 8)
        z = zeros[:, g:g + 1].astype(np.float64)
        q = np.where(s[:, None] > 0, np.rint(v / safe[:, None]), 0) + z
        codes[:, g * group:(g + 1) * group] = np.clip(q, 0, 15)
        scales[:, g] = s
    return codes, scales, zeros


def values(codes, scales, zeros, group):
    K = codes.shape[-1]
    spread = lambda a: np.repeat(np.asarray(a, np.float64), group, axis=-1)[..., :K]  # noqa: E731
    z = 8.0 if zeros is None else spread(zeros)
    return (codes.astype(np.float64) - z) * spread(scales)


def product(x, w, dx=0.0, terms=1):
    """(x w^T, bound): x within dx of what the kernel takes, cut into ``terms`` planes."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    K = w.shape[1]
    steps = -(-K // 16) * terms + -(-K // 32) + 16
    ref = x @ w.T
    size = np.abs(x) @ np.abs(w).T
    return ref, steps * STEP * size + np.broadcast_to(dx, x.shape) @ np.abs(w).T


def gated_mlp(x, gate, up, down, fp32=False):
    """(down(silu(gate x) * (up x)), bound).  Weights may come in two terms."""
    t, th = (3, 3) if fp32 else (2, 2)
    dx = np.abs(np.asarray(x, np.float64)) * (2.0 ** -24 if fp32 else 0.0)
    (g, dg), (u, du) = product(x, gate, dx, t), product(x, up, dx, t)
    s = g / (1 + np.exp(-g))
    h = s * u
    # |silu'| <= 1.1; the kernel's exp and division are within a few 2^-23
    # h in th terms of 8 bits, and (in two) the product of the two low terms left out
    dh = 1.1 * dg * (np.abs(u) + du) + np.abs(s) * du + np.abs(h) * (8 * STEP + 2.0 * 2.0 ** (-8 * th))
    return product(h, down, dh, 3)


def rounded(ref, bound, dtype):
    """The bound of the output after its rounding to ``dtype`` ("bfloat16", "float32")."""
    return bound + U[dtype] * (np.abs(ref) + bound)


def topk(logits, k, norm):
    """(ids, weights) of softmax's k largest, the lower expert among equals."""
    lg = np.asarray(logits, np.float64)
    p = np.exp(lg - lg.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    ids = np.argsort(-lg, axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(p, ids, 1)
    return ids, w / w.sum(1, keepdims=True) if norm else w


def moe(x, ids, weights, experts, fp32=False):
    """(sum_j w_j expert_{ids_j}(x), bound); experts: list of (gate, up, down) in float64,
    ids outside the list are dropped."""
    x = np.asarray(x, np.float64)
    out = np.zeros((x.shape[0], experts[0][2].shape[0]))
    bound, size = np.zeros_like(out), np.zeros_like(out)
    for e in range(len(experts)):
        t, j = np.nonzero(np.asarray(ids) == e)
        if len(t):
            y, dy = gated_mlp(x[t], *experts[e], fp32=fp32)
            w = np.asarray(weights, np.float64)[t, j][:, None]
            np.add.at(out, t, w * y)
            np.add.at(bound, t, np.abs(w) * dy)
            np.add.at(size, t, np.abs(w) * (np.abs(y) + dy))
    # weights are fp32 products, a token's terms are added in up to 8 + k partial sums
    return out, bound + (ids.shape[1] + 16) * STEP * size


def planes(v, count):
    """fp32 values cut into ``count`` bf16 terms, the rest dropped: their sum, as float64."""
    rest, total = np.asarray(v, np.float64), 0.0
    for _ in range(count):
        term = bf16(rest.astype(np.float32))
        total, rest = total + term, rest - term
    return total
