"""What the exact checks of ``test_few_precision_gpu.py`` see: mistakes planted in the restatement."""

from __future__ import annotations

import numpy as np
import pytest

import few_exact as fx
from oracle import group4 as og


def wrong(got, want):
    return float(np.mean(np.asarray(got) != np.asarray(want)))


def test_planes_hold_what_they_should():
    v = fx.fp32_values(1000, 0)
    assert wrong(og.planes(v, 3), v) == 0                  # 24 bits
    h = fx.products16(1000, 1)
    assert wrong(og.planes(h, 2), h) == 0                  # 16 bits
    w = fx.weights12(1000, 2)[0]
    assert wrong(og.planes(w, 2), w) == 0                  # a code's 5 bits times a scale's 8


@pytest.mark.parametrize("values,count", [(fx.fp32_values, 3), (fx.products16, 2)])
def test_a_missing_plane_is_seen(values, count):
    v = values(1000, 3)
    assert wrong(og.planes(v, count - 1), v) > 0.9


def test_a_missing_low_term_of_the_weights_is_seen():
    w, x = fx.weights12(4000, 4)[0], fx.bf16_values(4000, 5)
    # of the 15 codes, +-3, +-5, +-6 and +-7 times an odd scale of 8 bits have more than 8: 8 / 15
    assert wrong(x * og.planes(w, 1), x * w) > 0.5
    assert wrong((x * w).astype(np.float32).astype(np.float64), x * w) == 0
