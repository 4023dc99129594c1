"""Argument checks of the 4-bit weights and the few-token layer, and their CPU restatement (no GPU)."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from oracle import group4 as og
from sb200 import _lib, group4

P = 4096  # an aligned non-null pointer that a refused call never reads


def refused(rc, *words):
    assert rc < 0
    message = _lib.last_error()
    assert all(w in message for w in words), message


def matrix(**kw):
    return _lib.Group4(**{**dict(data=P, K=128, N=64, count=1, group=64, zeros=0), **kw})


def linear(m, x=P, xd=1, ldx=128, M=4, y=P, yd=1, ws=P, nb=1 << 30):
    return _lib.load().sb_group4_linear(x, xd, ldx, M, C.byref(m) if m else None, None, y, yd, ws, nb, None)


@pytest.mark.parametrize("field,value,word", [("K", 0, "positive"), ("N", -1, "positive"), ("K", 16385, "16384"), ("N", 1 << 25, "2^24"),
                                              ("group", 48, "group"), ("data", None, "null"), ("count", 0, "positive"),
                                              ("data", P + 8, "aligned")])
def test_matrix_refusals(field, value, word):
    refused(linear(matrix(**{field: value})), word)
    refused(_lib.load().sb_group4_dequantize(C.byref(matrix(**{field: value})), P, 0, None), word)


def test_linear_refusals():
    m = matrix()
    refused(linear(None), "null")
    refused(linear(m, xd=2), "x dtype")
    refused(linear(m, yd=7), "y dtype")
    refused(linear(m, M=-1), "tokens")
    refused(linear(m, M=(1 << 20) + 1), "tokens")
    refused(linear(matrix(count=2)), "one matrix")
    refused(linear(m, x=None), "x is null")
    refused(linear(m, y=None), "y is null")
    refused(linear(m, ldx=127), "overlap")
    assert linear(m, xd=0, ws=P, nb=16) == -6
    assert linear(m, x=P + 2, ws=None, nb=0) == -6
    assert linear(m, M=1 << 20, ws=None, nb=0) == -6  # (so many that the weights are written out)
    refused(linear(m, xd=0, ws=P + 16), "aligned")
    assert linear(m, M=0, x=None, y=None, ws=None, nb=0) == 0


def test_quantize_and_pack_refusals():
    lib = _lib.load()
    q = lambda w=P, wd=0, ldw=128, **kw: lib.sb_group4_quantize(w, wd, ldw, C.byref(matrix(**kw)), None, None)  # noqa: E731
    refused(q(w=None), "null")
    refused(q(wd=2), "dtype")
    refused(q(ldw=100), "stride")
    refused(q(group=16), "group")
    refused(q(K=0), "positive")
    refused(q(data=None), "null")
    p = lambda codes=P, scales=P, zeros=None, **kw: lib.sb_group4_pack(codes, scales, zeros, C.byref(matrix(**kw)), None)  # noqa: E731
    refused(p(codes=None), "null")
    refused(p(scales=None), "null")
    refused(p(zeros=P), "zero points")
    refused(p(N=0), "positive")
    assert lib.sb_group4_matrix_bytes(129, 17, 32, 1) == 2 * 2 * (1024 + 4 * 48)
    assert lib.sb_group4_matrix_bytes(128, 16, 128, 0) == 1024 + 32
    assert lib.sb_group4_matrix_bytes(0, 3, 32, 0) == 0 and lib.sb_group4_matrix_bytes(8, 3, 33, 0) == 0


def test_ternary_pack_refusals():
    lib = _lib.load()
    refused(lib.sb_ternary_pack(None, 4, 4, P, None), "null")
    refused(lib.sb_ternary_pack(P, 0, 4, P, None), "positive")


def test_gated_mlp_refusals():
    lib = _lib.load()

    def call(gate, up, down, xd=1, ldx=128, M=3, yd=1, nb=1 << 30):
        return lib.sb_group4_gated_mlp(P, xd, ldx, M, C.byref(gate), C.byref(up), C.byref(down), P, yd, P, nb, None)

    g, d = matrix(), matrix(K=64, N=128)
    refused(call(g, matrix(N=32), d), "same shape")
    refused(call(g, matrix(group=32), d), "same shape")
    refused(call(g, matrix(zeros=1), d), "zero points")
    refused(call(g, g, g), "down must be")
    refused(call(g, g, d, xd=3), "x dtype")
    refused(call(g, g, d, yd=3), "y dtype")
    refused(call(g, g, d, ldx=2), "overlap")
    assert call(g, g, d, nb=8) == -6
    assert call(g, g, d, M=0) == 0


def test_moe_few_refusals():
    lib = _lib.load()

    def call(B=2, k=2, gate=None, gd=1, xd=1, od=0, ldx=128, ids=P, w=P, out=P, nb=1 << 30, **kw):
        ex = _lib.Experts(**{**dict(kind=1, n_experts=8, hidden=128, intermediate=64, group=64, gate=P, up=P, down=P,
                                    gate_scale=P, up_scale=P, down_scale=P, zeros=0), **kw})
        return lib.sb_moe_few(C.byref(ex), P, xd, ldx, B, k, gate, gd, 0, ids, w, out, od, P, nb, None)

    refused(call(hidden=0), "H=0")
    refused(call(hidden=8193, ldx=8193), "8192")
    refused(call(intermediate=8193), "8192")
    refused(call(n_experts=0), "experts")
    refused(call(n_experts=513), "experts")
    refused(call(k=0), "top_k")
    refused(call(k=33), "top_k")
    refused(call(k=9, gate=P), "top_k 9 of 8")
    refused(call(B=257), "tokens")
    refused(call(B=65, k=32), "tokens")
    refused(call(B=-1), "tokens")
    refused(call(kind=2), "kind")
    refused(call(group=96), "group")
    refused(call(kind=0, gate_scale=None), "null expert")
    refused(call(up=None), "null expert")
    refused(call(down=P + 8), "aligned")
    refused(call(xd=2), "x dtype")
    refused(call(od=2), "out dtype")
    refused(call(gate=P, gd=2), "gate dtype")
    refused(call(ids=None), "null ids")
    refused(call(out=None), "null ids")
    refused(call(ldx=5), "overlap")
    assert call(nb=0) == -6
    assert call(B=0) == 0
    assert [lib.sb_moe_few_max_tokens(k) for k in (0, 1, 8, 9, 32, 33)] == [0, 256, 256, 227, 64, 0]
    refused(lib.sb_moe_few(None, P, 1, 128, 1, 1, None, 1, 0, P, P, P, 0, P, 1 << 20, None), "null experts")


def test_python_refusals_without_a_gpu():
    """CPU tensors and wrong arguments raise before anything is launched."""
    from sb200.moe import FewTokenMoE
    x = torch.zeros(2, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        group4.quantize(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        group4.Group4Matrix.pack(torch.zeros(2, 128, dtype=torch.uint8), torch.ones(2, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        group4.Group4Matrix(torch.zeros(1056, dtype=torch.uint8), 2, 128, 128, False)
    with pytest.raises(RuntimeError, match="group"):
        group4.Group4Matrix(torch.zeros(1056, dtype=torch.uint8), 2, 128, 100, False)

    class E:
        E, H, gate = 4, 128, x

    with pytest.raises(RuntimeError, match="gate_weight"):
        FewTokenMoE(E, torch.zeros(3, 128))
    with pytest.raises(RuntimeError, match="top_k"):
        FewTokenMoE(E, torch.zeros(4, 128), top_k=5)
    with pytest.raises(RuntimeError, match="dtype"):
        FewTokenMoE(E, torch.zeros(4, 128, dtype=torch.float16), top_k=2)


def test_restated_quantiser():
    """By hand: one group, symmetric and not, a tie and a zero row."""
    w = np.array([[7.0, -7.0, 0.5, 1.5, 2.5, -0.5], [0, 0, 0, 0, 0, 0]])
    codes, scales, zeros = og.quantize(w, 32)
    assert scales.tolist() == [[1.0], [0.0]]
    assert codes.tolist() == [[15, 1, 8, 10, 10, 8], [8] * 6]
    codes, scales, zeros = og.quantize(np.array([[-1.0, 14.0, 0.0, 0.5]]), 32, symmetric=False)
    assert (scales, zeros) == ([[1.0]], [[1]]) and codes.tolist() == [[0, 15, 1, 1]]
    v = og.values(codes, scales, zeros, 32)
    assert v.tolist() == [[-1.0, 14.0, 0.0, 0.0]]


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_scales_of_data_inside_a_larger_buffer(group, zeros):
    """Scales and zero points are read from the matrix's own bytes, wherever they begin."""
    N, K, count = 33, 300, 2
    nbytes = count * _lib.load().sb_group4_matrix_bytes(K, N, group, int(zeros))
    data = torch.from_numpy(np.random.default_rng(group).integers(0, 256, nbytes).astype(np.uint8))

    def matrix_on(d):
        m = group4.Group4Matrix.__new__(group4.Group4Matrix)
        m.N, m.K, m.group, m.count, m.has_zeros, m.data = N, K, group, count, zeros, d
        return m

    buffer = torch.zeros(nbytes + 4096, dtype=torch.uint8)
    buffer[1040:1040 + nbytes] = data
    whole, part = matrix_on(data), matrix_on(buffer[1040:1040 + nbytes])
    assert torch.equal(part.scales.view(torch.int16), whole.scales.view(torch.int16))
    # row 17 = 16 + 1 of the second matrix: tile 1, place 2 of each group's scales (after 1024 bytes of words)
    block, per = 1024 + (48 if zeros else 32) * (128 // group), 128 // group
    at = ((1 * 3 + 1) * 3 + 0) * block + 1024 + 2 * 2
    assert part.scales[N + 17, 0].view(torch.int16) == data[at:at + 2].view(torch.int16)[0]
    if zeros:
        assert torch.equal(part.zeros, whole.zeros)
        assert part.zeros[N + 17, 0] == data[((1 * 3 + 1) * 3) * block + 1024 + 32 * per + 2]
    else:
        assert part.zeros is None


def test_experts_past_the_layers_limits_are_refused_when_made():
    """Not at the first call, when the weights have been packed; the limits are the kernels' own."""
    from types import SimpleNamespace

    from sb200.moe import FewTokenMoE
    E, W = group4.MAX_EXPERTS, group4.MAX_WIDTH

    def few(E, H, I):
        ex = _lib.Experts(kind=1, n_experts=E, hidden=H, intermediate=I, group=64, gate=P, up=P, down=P, zeros=0)
        return _lib.load().sb_moe_few(C.byref(ex), P, 1, H, 0, 1, None, 1, 0, P, P, P, 0, P, 1 << 30, None)

    assert few(E, W, W) == 0
    data = torch.empty(0)
    for e, h, i in ((E + 1, 64, 32), (4, W + 1, 32), (4, 64, W + 1)):
        refused(few(e, h, i))
        mats = [SimpleNamespace(count=e, N=n, K=k, group=64, has_zeros=False, device=data.device, data=data)
                for n, k in ((i, h), (i, h), (h, i))]
        with pytest.raises(RuntimeError, match="up to 512 experts and 8192"):
            group4.Group4Experts(*mats)
        on_cpu = [torch.empty(e, n, k, device="meta", dtype=torch.uint8) for n, k in ((i, h), (i, h), (h, i))]
        with pytest.raises(RuntimeError, match="up to 512 experts and 8192"):
            group4.Group4Experts.quantize(*on_cpu)
        with pytest.raises(RuntimeError, match="up to 512 experts and 8192"):
            group4.Group4Experts.pack(*({"codes": t, "scales": t} for t in on_cpu))
        with pytest.raises(RuntimeError, match="up to 512 experts and 8192"):
            FewTokenMoE(SimpleNamespace(E=e, H=h, I=i, gate=data), torch.empty(e, h), top_k=1)
    mats = [SimpleNamespace(count=E, N=W, K=W, group=64, has_zeros=False, device=data.device, data=data) for _ in range(3)]
    assert group4.Group4Experts(*mats).E == E


def test_which_form_a_batch_takes():
    """An empty batch is no few-token batch: with few_tokens off nothing goes to forward_few, whose
    limits are narrower; tokens are counted by their routing."""
    from sb200.moe import BVHMoELayer
    from sb200.ternary import TernaryExperts

    class Experts(TernaryExperts):
        def __init__(self):
            pass

        def forward(self, x, ids, w, out_dtype=None, out=None):
            return "grouped"

        def forward_few(self, x, ids, w, out_dtype=None, out=None):
            return "few"

    def runs(few_tokens, B, lead=()):
        layer = BVHMoELayer(None, Experts(), device="cpu", few_tokens=few_tokens)
        return layer.forward_topk(torch.zeros(*(lead or (B,)), 4), torch.zeros(B, 40), torch.zeros(B, 40, dtype=torch.int32))

    assert [runs(0, B) for B in (0, 1, 300)] == ["grouped"] * 3
    assert [runs(16, B) for B in (0, 1, 16, 17)] == ["grouped", "few", "few", "grouped"]
    assert runs(16, 24, lead=(2, 12)) == "grouped"


def test_overlap():
    """Where two views of one storage meet, and where they only lie side by side."""
    b = torch.zeros(100)
    f = group4._overlap
    assert f(b[:10], b[9:12]) and f(b[9:12], b[:10]) and f(b, b[50:51]) and f(b[50:51], b)
    assert not f(b[:10], b[10:12]) and not f(b[10:12], b[:10])
    assert not f(b[:10], torch.zeros(10)) and not f(b[:0], b) and not f(b, b[5:5])
    rows = b[:96].view(12, 8)
    assert f(rows[:, :4], b[4:5]) and not f(rows[:6], rows[6:]) and f(rows[:, 1], b[9:10])
    assert f(b[:10], b.view(torch.int32)[9:11]) and not f(b[:10], b.view(torch.int16)[20:22])
    assert f(b[3:4].expand(5), b[3:4]) and not f(b[3:4].expand(5), b[4:5])
