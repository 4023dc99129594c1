"""Products whose results are exact in fp32, for checks without a tolerance: every output is one
product, all other weights are zero, and the values have as many bits as the kernels say they
keep."""

from __future__ import annotations

import numpy as np

from oracle import group4 as og


def _signed(rng, lo, hi, n, step):
    """Odd multiples of ``step`` with magnitudes in [lo, hi): every bit down to the step counts."""
    k = rng.integers(round(lo / step), round(hi / step), n) | 1
    return k * step * rng.choice([-1.0, 1.0], n)


def fp32_values(n, seed):
    """24 significant bits, the last one set."""
    return _signed(np.random.default_rng(seed), 1.0, 2.0, n, 2.0 ** -23)


def bf16_values(n, seed):
    """8 significant bits, the last one set."""
    return _signed(np.random.default_rng(seed), 1.0, 2.0, n, 2.0 ** -7)


def products16(n, seed):
    """Products of two values of 8 significant bits."""
    return bf16_values(n, seed) * bf16_values(n, seed + 1000)


def weights12(n, seed):
    """(values, codes, scales): code - 8 times a bf16 scale of 8 significant bits."""
    rng = np.random.default_rng(seed)
    codes = rng.choice([0, 1, 2, 3, 4, 5, 6, 7, 9, 10, 11, 12, 13, 14, 15], n)
    scales = np.abs(bf16_values(n, seed + 2000))
    return (codes - 8.0) * scales, codes.astype(np.uint8), scales


def selection(N, K, seed, group=None):
    """A matrix with one weight in each row: (columns [N], codes uint8 [N, K] of 8 but there, scales
    [N, groups], values [N] of the weights).  Without a group the weights are 1 and -1 at scale 1."""
    rng = np.random.default_rng(seed)
    at = rng.integers(0, K, N)
    at[: min(N, 2)] = [0, K - 1][: min(N, 2)]
    codes = np.full((N, K), 8, np.uint8)
    if group is None:
        w, c, s = rng.choice([-1.0, 1.0], N), None, np.ones(N)
        c = (8 + w).astype(np.uint8)
    else:
        w, c, s = weights12(N, seed)
    codes[np.arange(N), at] = c
    scales = np.repeat(s[:, None], -(-K // (group or 32)), 1)
    return at, codes, og.bf16(scales), w
