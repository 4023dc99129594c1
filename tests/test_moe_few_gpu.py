"""The few-token MoE layer against the float64 restatement (needs a B200)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import group4 as og
from test_group4_gpu import acts, close

pytestmark = pytest.mark.gpu


def make_experts(kind, E, H, I, device, group=64, zeros=True, seed=0):
    """(experts, [(gate, up, down) float64 per expert])."""
    from sb200 import group4
    from sb200.ternary import TernaryExperts
    rng = np.random.default_rng(seed)
    shapes = [(I, H), (I, H), (H, I)]
    to = lambda a: torch.from_numpy(a).to(device)  # noqa: E731
    if kind == "ternary":
        t = [rng.integers(-1, 2, (E, n, k)).astype(np.int8) for n, k in shapes]
        s = [(rng.uniform(0.5, 1.5, (E, n)) / np.sqrt(k)).astype(np.float32) for n, k in shapes]
        vals = [a.astype(np.float64) * b.astype(np.float64)[..., None] for a, b in zip(t, s)]
        return TernaryExperts.from_tensors(*map(to, t), *map(to, s)), list(zip(*vals))
    ms, vals = [], []
    for n, k in shapes:
        G = -(-k // group)
        codes = rng.integers(0, 16, (E, n, k)).astype(np.uint8)
        scales = og.bf16(rng.uniform(0.5, 1.5, (E, n, G)) / np.sqrt(k) / 4)
        z = rng.integers(0, 16, (E, n, G)).astype(np.uint8) if zeros else None
        ms.append({"codes": to(codes), "scales": to(scales), "zeros": None if z is None else to(z)})
        vals.append(og.values(codes, scales, z, group))
    return group4.Group4Experts.pack(*ms, group=group), list(zip(*vals))


def routing(B, k, E, seed):
    rng = np.random.default_rng(seed)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(B)]).astype(np.int32)
    return ids, rng.uniform(0.05, 1.0, (B, k)).astype(np.float32)


def reference(x, ids, w, vals):
    return og.moe(x.double().cpu().numpy(), np.asarray(ids), np.asarray(w), vals, fp32=x.dtype == torch.float32)


@pytest.mark.parametrize("kind", ["ternary", "group4"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,E,k,H,I", [(1, 8, 2, 256, 128), (1, 64, 8, 512, 256), (3, 5, 5, 72, 40), (8, 16, 4, 130, 33),
                                       (9, 4, 1, 264, 96), (31, 3, 2, 100, 65), (64, 16, 4, 256, 128), (200, 2, 1, 64, 16),
                                       (256, 7, 7, 40, 24), (2, 1, 1, 1, 1), (5, 300, 3, 16, 8), (128, 4, 1, 64, 100),
                                       (100, 3, 1, 33, 16), (64, 512, 32, 8192, 8), (9, 512, 32, 8, 8192)])
def test_given_routing(cuda_device, kind, dtype, B, E, k, H, I):
    ex, vals = make_experts(kind, E, H, I, cuda_device, seed=E)
    x = acts(B, H, dtype, cuda_device, seed=B)
    ids, w = routing(B, k, E, seed=B)
    y = ex.forward_few(x, torch.from_numpy(ids).to(cuda_device), torch.from_numpy(w).to(cuda_device))
    assert y.dtype == torch.float32 and y.shape == (B, H)
    ref, bound = reference(x, ids, w, vals)
    close(y, ref, bound, kind)


@pytest.mark.parametrize("kind", ["ternary", "group4"])
@pytest.mark.parametrize("B,E,k,H,I", [(250, 300, 1, 48, 16), (256, 2, 2, 64, 2100), (256, 40, 8, 2056, 24)])
def test_uneven_groups(cuda_device, kind, B, E, k, H, I):
    """Most tokens at a few experts, one or two at many: groups of every size, a unit or many to each."""
    ex, vals = make_experts(kind, E, H, I, cuda_device, seed=E)
    rng = np.random.default_rng(B)
    few = np.stack([rng.permutation(min(E, k + 1))[:k] for _ in range(B)])
    ids = np.where(rng.random((B, 1)) < 0.6, few, np.stack([rng.permutation(E)[:k] for _ in range(B)])).astype(np.int32)
    w = rng.uniform(0.1, 1, (B, k)).astype(np.float32)
    x = acts(B, H, torch.bfloat16, cuda_device, seed=I)
    y = ex.forward_few(x, torch.from_numpy(ids).to(cuda_device), torch.from_numpy(w).to(cuda_device))
    ref, bound = reference(x, ids, w, vals)
    close(y, ref, bound, kind)


@pytest.mark.parametrize("kind", ["ternary", "group4"])
@pytest.mark.parametrize("dtype,gate_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                              (torch.float32, torch.float32)])
@pytest.mark.parametrize("B,E,k,H,I,norm", [(1, 64, 8, 256, 64, False), (6, 8, 8, 130, 40, True), (33, 40, 3, 128, 48, False),
                                            (70, 300, 5, 64, 16, True), (256, 16, 8, 32, 16, False)])
def test_with_gate(cuda_device, kind, dtype, gate_dtype, B, E, k, H, I, norm):
    from sb200.moe import FewTokenMoE
    ex, vals = make_experts(kind, E, H, I, cuda_device, seed=E + 1)
    x = acts(B, H, dtype, cuda_device, seed=B)
    gw = (acts(E, H, torch.float32, cuda_device, seed=77) / H ** 0.5).to(gate_dtype)
    layer = FewTokenMoE(ex, gw, top_k=k, norm_topk=norm)
    y, ids, w = layer(x, routing=True)
    assert y.dtype == dtype and ids.dtype == torch.int32
    logits = (x.double().cpu() @ gw.double().cpu().t()).float().double().numpy()
    rid, rw = og.topk(logits, k, norm)
    np.testing.assert_array_equal(ids.cpu().numpy(), rid)
    # exp within 2 ulp of an argument that is within half an ulp, sums of E terms, two divisions
    spread = np.abs(logits - logits.max(1, keepdims=True)).max()
    np.testing.assert_allclose(w.double().cpu().numpy(), rw, rtol=(spread + E + k + 8) * 2.0 ** -24 * 2)
    ref, bound = reference(x, rid, w.cpu().numpy(), vals)
    close(y, ref, bound, kind)
    assert torch.equal(y, layer(x))


def test_equal_and_non_finite_logits(cuda_device):
    """Ties go to the lower expert; NaN and -inf logits rank last, NaN makes the token NaN."""
    from sb200 import _lib
    from sb200.moe import FewTokenMoE
    E, H, k = 40, 64, 6
    ex, _ = make_experts("group4", E, H, 32, cuda_device)
    gw = torch.zeros(E, H, device=cuda_device)
    x = torch.ones(4, H, device=cuda_device)
    y, ids, w = FewTokenMoE(ex, gw, k)(x, routing=True)
    assert (ids.cpu() == torch.arange(k, dtype=torch.int32)).all()
    np.testing.assert_allclose(w.cpu().numpy(), 1 / E, rtol=2.0 ** -20)
    gw[:, 0] = -torch.inf
    gw[7, 0] = gw[21, 0] = 1.0
    y, ids, w = FewTokenMoE(ex, gw, k)(x, routing=True)
    assert ids[0].tolist() == [7, 21, 0, 1, 2, 3]
    assert torch.equal(w[0].cpu(), torch.tensor([0.5, 0.5, 0, 0, 0, 0])) and y.isfinite().all()
    gw[3, 0] = torch.nan
    y, ids, w = FewTokenMoE(ex, gw, k)(x, routing=True)
    assert ids[0].tolist() == [7, 21, 0, 1, 2, 3] and w.isnan().all() and y.isnan().all()
    torch.cuda.synchronize()
    assert _lib.load().sb_device_status(0) == -1 and "non-finite" in _lib.last_error()


@pytest.mark.parametrize("kind", ["ternary", "group4"])
def test_dropped_and_repeated_ids(cuda_device, kind):
    from sb200 import _lib
    ex, vals = make_experts(kind, 6, 96, 48, cuda_device)
    x = acts(5, 96, torch.bfloat16, cuda_device)
    w = np.random.default_rng(0).uniform(0.1, 1, (5, 4)).astype(np.float32)
    ids = np.array([[2, 2, 2, 2], [0, 1, 0, 5], [-1, 6, 3, 3], [-1, -7, 99, 2 ** 31 - 1], [4, 3, 2, 1]], np.int32)
    y = ex.forward_few(x, torch.from_numpy(ids).to(cuda_device), torch.from_numpy(w).to(cuda_device))
    torch.cuda.synchronize()
    assert _lib.load().sb_device_status(0) == -1 and "expert id" in _lib.last_error()
    ref, bound = reference(x, ids, w, vals)
    close(y, ref, bound, kind)
    assert (y[3] == 0).all()


def test_id_types_and_refusals(cuda_device):
    from sb200 import _lib
    from sb200.moe import FewTokenMoE
    ex, _ = make_experts("group4", 6, 96, 48, cuda_device)
    x = acts(5, 96, torch.bfloat16, cuda_device)
    ids, w = (torch.from_numpy(a).to(cuda_device) for a in routing(5, 2, 6, seed=3))
    want = ex.forward_few(x, ids, w)
    for t in (torch.int64, torch.int16, torch.uint8):
        assert torch.equal(ex.forward_few(x, ids.to(t), w), want)
    assert torch.equal(ex.forward_few(x, ids.t().contiguous().t(), w.double()), want)
    far = ids.long()
    far[0] = torch.tensor([2 ** 32 + 1, -2 ** 40], device=cuda_device)  # would be 1 and 0 in 32 bits
    y = ex.forward_few(x, far, w)
    torch.cuda.synchronize()
    assert _lib.load().sb_device_status(0) == -1 and (y[0] == 0).all() and torch.equal(y[1:], want[1:])
    for bad in ((x, ids.float(), w), (x, ids[:4], w), (x, ids, w[:, :1]), (x, ids.cpu(), w), (x[:, :95], ids, w),
                (x.half(), ids, w)):
        with pytest.raises(RuntimeError):
            ex.forward_few(*bad)
    with pytest.raises(RuntimeError, match="overlaps"):
        ex.forward_few(x, ids, w, out=x)
    with pytest.raises(RuntimeError, match="gate_weight"):
        FewTokenMoE(ex, torch.zeros(6, 95, device=cuda_device), 2)


@pytest.mark.parametrize("N,K", [(1, 1), (5, 63), (16, 64), (7, 200), (33, 1000)])
def test_ternary_pack_equals_the_host_packer(cuda_device, N, K):
    from sb200 import ternary
    t = torch.from_numpy(np.random.default_rng(K).integers(-1, 2, (2, N, K)).astype(np.int8)).to(cuda_device)
    got = ternary._pack(t.reshape(2 * N, K))
    np.testing.assert_array_equal(got.cpu().numpy().view(np.uint32), ternary.pack_device(t.cpu().numpy().reshape(2 * N, K)))


def test_agrees_with_the_grouped_layer(cuda_device):
    """forward_few and forward are the same sums in another order, at the layer's own sizes."""
    from sb200.ternary import TernaryExperts
    ex = TernaryExperts.random(64, 2048, 1024, 3, cuda_device)
    for B in (1, 24):
        x = acts(B, 2048, torch.bfloat16, cuda_device, seed=B)
        ids, w = (torch.from_numpy(a).to(cuda_device) for a in routing(B, 8, 64, seed=B))
        a, b = ex.forward(x, ids, w), ex.forward_few(x, ids, w)
        # the grouped layer's hidden state is fp16: 2^-11 each, averaged over 1024 channels
        assert float((a - b).norm() / a.norm()) < 2.0 ** -11


def test_batches_past_one_call(cuda_device):
    """Any batch: cut into calls whose tokens do not depend on the cut."""
    from sb200 import group4
    from sb200.moe import FewTokenMoE
    ex, vals = make_experts("group4", 8, 64, 32, cuda_device)
    gw = acts(8, 64, torch.float32, cuda_device, seed=5)
    most = group4.max_tokens(3)
    assert most == 256
    x = acts(2 * most + 37, 64, torch.bfloat16, cuda_device)
    layer = FewTokenMoE(ex, gw, 3)
    y, ids, w = layer(x, routing=True)
    ref, bound = reference(x, ids.cpu().numpy(), w.cpu().numpy(), vals)
    close(y, ref, bound)
    assert layer(x[:0]).shape == (0, 64)
    assert ex.forward_few(x[:0], ids[:0], w[:0]).shape == (0, 64)
    y3 = layer(x[:24].view(2, 3, 4, 64))
    assert y3.shape == (2, 3, 4, 64) and torch.equal(y3.view(24, 64), layer(x[:24]))


@pytest.mark.parametrize("kind", ["ternary", "group4"])
def test_non_finite_tokens_stay_alone(cuda_device, kind):
    from sb200 import _lib
    ex, _ = make_experts(kind, 4, 128, 64, cuda_device)
    for dtype in (torch.bfloat16, torch.float32):
        x = acts(20, 128, dtype, cuda_device)
        ids, w = (torch.from_numpy(a).to(cuda_device) for a in routing(20, 2, 4, seed=1))
        clean = ex.forward_few(x, ids, w)
        x[6, 3], x[11] = torch.nan, torch.inf
        y = ex.forward_few(x, ids, w)
        keep = torch.ones(20, dtype=torch.bool, device=cuda_device)
        keep[6] = keep[11] = False
        assert torch.equal(y[keep], clean[keep]) and not y[6].isfinite().any() and not y[11].isfinite().any()
        torch.cuda.synchronize()
        assert _lib.load().sb_device_status(0) == -1


def test_layer_paths(cuda_device):
    """BVHMoELayer: few_tokens sends small batches to forward_few and leaves larger ones
    as they were; 4-bit experts serve behind the same router; the graph replays both."""
    from sb200.moe import BVHMoELayer, GraphedLayer
    from test_moe_layer_gpu import make_layer
    layer, experts = make_layer(cuda_device)
    few = BVHMoELayer(layer.router, layer.experts, top_k=4, few_tokens=16)
    for B in (1, 16, 17):
        x = acts(B, 256, torch.bfloat16, cuda_device, seed=B)
        ids, w = layer.route(x)
        want = layer.experts.forward_few if B <= 16 else layer.experts.forward
        assert torch.equal(few(x), want(x, ids, w, out_dtype=x.dtype))
        assert torch.equal(few.forward_topk(x, w, ids), want(x, ids, w, out_dtype=x.dtype))
    e4, vals = make_experts("group4", 16, 256, 128, cuda_device)
    l4 = BVHMoELayer(layer.router, e4, top_k=4)
    for B in (2, 600):
        x = acts(B, 256, torch.bfloat16, cuda_device, seed=B)
        ids, w = l4.route(x)
        ref, bound = reference(x, ids.cpu().numpy(), w.cpu().numpy(), vals)
        close(l4(x), ref, bound)
    x, out = acts(3, 256, torch.bfloat16, cuda_device), torch.empty(3, 256, dtype=torch.bfloat16, device=cuda_device)
    for layer_ in (few, l4):
        graphed = GraphedLayer(layer_)
        graphed(x, out)
        first = out.clone()
        assert torch.equal(first, layer_(x))
        x.mul_(0.5)
        graphed(x, out)
        assert torch.equal(out, layer_(x)) and not torch.equal(out, first)


def test_quantised_layer_as_it_is_used(cuda_device):
    """Float experts quantised to 4 bits, one token after another through a graph on a side
    stream, then a prompt: the operators together."""
    from sb200 import group4
    from sb200.moe import FewTokenMoE
    E, H, I, k = 12, 192, 96, 3
    g = torch.Generator().manual_seed(0)
    ws = [torch.randn(E, n, c, generator=g).to(cuda_device) / c ** 0.5 for n, c in ((I, H), (I, H), (H, I))]
    gw = torch.randn(E, H, generator=g).to(cuda_device) / H ** 0.5
    ex = group4.Group4Experts.quantize(*ws, group=32, symmetric=False)
    vals = list(zip(*(m.dequantize().double().cpu().numpy().reshape(E, -1, m.K) for m in (ex.gate, ex.up, ex.down))))
    layer = FewTokenMoE(ex, gw, k, norm_topk=True)
    x = acts(1, H, torch.bfloat16, cuda_device)
    y = torch.empty_like(x)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _, ids, w = layer(x, out=y, routing=True)
    side.synchronize()
    for step in range(4):
        x.copy_(acts(1, H, torch.bfloat16, cuda_device, seed=step))
        graph.replay()
        ref, bound = reference(x, ids.cpu().numpy(), w.cpu().numpy(), vals)
        close(y, ref, bound, f"step {step}")
        assert torch.equal(y, layer(x))
    prompt = acts(300, H, torch.bfloat16, cuda_device, seed=9)
    yp, ids, w = layer(prompt, routing=True)
    ref, bound = reference(prompt, ids.cpu().numpy(), w.cpu().numpy(), vals)
    close(yp, ref, bound, "prompt")


def test_gate_that_needs_a_gradient_is_refused(cuda_device):
    """A trained gate (an nn.Linear's weight) gets no gradient here: outside no_grad it raises."""
    from sb200.moe import FewTokenMoE
    ex, _ = make_experts("group4", 6, 96, 48, cuda_device)
    gate = torch.nn.Linear(96, 6, bias=False, device=cuda_device)
    x = acts(3, 96, torch.bfloat16, cuda_device)
    layer = FewTokenMoE(ex, gate.weight, 2)
    with pytest.raises(RuntimeError, match="gradient"):
        layer(x)
    with torch.no_grad():
        y = layer(x)
    assert torch.equal(y, FewTokenMoE(ex, gate.weight.detach(), 2)(x))


def test_gate_is_read_at_each_call(cuda_device):
    """A gate whose rows are not contiguous is no snapshot, and one that has changed its
    device, shape or dtype since the layer was made is refused."""
    from sb200.moe import FewTokenMoE
    ex, _ = make_experts("group4", 6, 96, 48, cuda_device)
    x = acts(3, 96, torch.bfloat16, cuda_device)
    for gate in (acts(96, 6, torch.float32, cuda_device, seed=3).t(), acts(6, 200, torch.float32, cuda_device, seed=3)[:, :96]):
        layer = FewTokenMoE(ex, gate, 2)
        assert torch.equal(layer(x), FewTokenMoE(ex, gate.contiguous(), 2)(x))
        gate.mul_(-1)
        assert torch.equal(layer(x), FewTokenMoE(ex, gate.contiguous(), 2)(x))
    linear = torch.nn.Linear(96, 6, bias=False, device=cuda_device).requires_grad_(False)
    layer = FewTokenMoE(ex, linear.weight, 2)
    layer(x)
    for change, word in ((lambda: linear.half(), "dtype"), (lambda: linear.cpu(), "CUDA"),
                         (lambda: linear.weight.set_(torch.zeros(5, 96, device=cuda_device)), "shape")):
        linear.to(cuda_device, torch.float32)
        change()
        with pytest.raises(RuntimeError, match=word):
            layer(x)


def test_out_that_overlaps_the_routing_or_the_gate_is_refused(cuda_device):
    from sb200.moe import FewTokenMoE
    ex, _ = make_experts("group4", 6, 96, 48, cuda_device)
    x = acts(3, 96, torch.bfloat16, cuda_device)
    ids, w = (torch.from_numpy(a).to(cuda_device) for a in routing(3, 2, 6, seed=3))
    buffer = torch.zeros(6 * 96 + 6, device=cuda_device)
    out, behind = buffer[:3 * 96].view(3, 96), buffer[6 * 96:].view(3, 2)
    inside = buffer[100:106].view(3, 2)
    for bad in ((inside.view(torch.int32), w), (ids, inside)):
        with pytest.raises(RuntimeError, match="overlaps"):
            ex.forward_few(x, *bad, out=out)
    with pytest.raises(RuntimeError, match="overlaps the gate"):
        FewTokenMoE(ex, buffer[:6 * 96].view(6, 96), 2)(x, out=out)
    behind.copy_(w)
    assert torch.equal(ex.forward_few(x, ids, behind, out=out), ex.forward_few(x, ids, w))
