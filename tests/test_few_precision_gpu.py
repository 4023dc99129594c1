"""The bits that the few-token kernels keep, without tolerances (needs a B200): products whose exact
results are fp32 numbers (``few_exact.py``), so that a lost plane of the activations or of the
hidden state, or a lost low term of the weights, shows in nearly every output."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import few_exact as fx

pytestmark = pytest.mark.gpu


def matrix(codes, scales, group, device):
    from sb200 import group4
    return group4.Group4Matrix.pack(torch.from_numpy(codes).to(device), torch.from_numpy(scales).to(device), group=group)


def dev(a, device, dtype=torch.float32):
    t = torch.from_numpy(np.ascontiguousarray(a))
    assert torch.equal(t.to(dtype).double(), t.double())
    return t.to(dtype).to(device)


def same(y, want):
    np.testing.assert_array_equal(y.double().cpu().numpy(), want)


@pytest.mark.parametrize("M,K,N", [(1, 2048, 777), (3, 1000, 130), (8, 129, 48), (17, 384, 100), (70, 264, 65), (300, 72, 33),
                                   (2, 16384, 40)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_linear_keeps_fp32_activations(cuda_device, M, K, N, group):
    """24 bits through a weight of 1 or -1; through a weight of 12, the product's one rounding."""
    x = fx.fp32_values(M * K, M).reshape(M, K)
    from sb200 import group4
    at, codes, scales, w = fx.selection(N, K, seed=N)
    scales = np.repeat(scales[:, :1], -(-K // group), 1)
    same(group4.linear(dev(x, cuda_device), matrix(codes, scales, group, cuda_device)), x[:, at] * w)
    # +-1 at a scale of 8 bits: the scaled sum is rounded once
    scales = np.repeat(np.abs(fx.bf16_values(N, 9))[:, None], -(-K // group), 1)
    y = group4.linear(dev(x, cuda_device), matrix(codes, scales, group, cuda_device))
    same(y, (x[:, at] * w * scales[:, 0]).astype(np.float32))


@pytest.mark.parametrize("M,K,N,long", [(1, 2048, 777, False), (9, 1000, 130, False), (16, 384, 100, False), (300, 72, 33, False),
                                        (1100, 130, 1024, True), (1300, 72, 1001, True), (200, 8184, 4100, True)])
@pytest.mark.parametrize("group", [32, 128])
def test_linear_keeps_the_weights(cuda_device, M, K, N, long, group):
    """bf16 activations times weights of 12 bits, in the short form and in the long one's two terms."""
    from sb200 import _lib, group4
    assert (_lib.load().sb_group4_linear_workspace_bytes(_lib.SB_BF16, M, K, N) > 2 * M * (-(-K // 8) * 8) + 255) is long
    x = fx.bf16_values(M * K, M).reshape(M, K)
    at, codes, scales, w = fx.selection(N, K, seed=N, group=group)
    y = group4.linear(dev(x, cuda_device, torch.bfloat16), matrix(codes, scales, group, cuda_device), out_dtype=torch.float32)
    same(y, x[:, at] * w)


def swiglu(H, I, seed, group, fp32, down_bits):
    """Gate, up and down whose hidden values are products: channel 0 of a token is 1, so that the gate
    is its weight, at least 32, where silu(g) = g in fp32; up selects a channel; down selects a
    hidden value, by 1 or -1 or a weight of 12 bits.  fp32: the gate is 32, and the hidden value
    keeps an activation's 24 bits; bf16: the gate has 8 bits, the hidden value 16 (8 behind a
    weight of 12).  Returns three (codes, scales) and f(x) = the layer's exact output."""
    g = np.full(I, 32.0) if fp32 or down_bits else 32 * np.abs(fx.bf16_values(I, seed))
    gate = np.full((I, H), 8, np.uint8)
    gate[:, 0] = 9
    groups = lambda K: -(-K // group)  # noqa: E731
    at, up, up_s, u = fx.selection(I, H, seed + 1)
    to, down, down_s, d = fx.selection(H, I, seed + 2, group if down_bits else None)
    spread = lambda s, K: np.repeat(s[:, :1], groups(K), 1)  # noqa: E731
    parts = ((gate, np.repeat(g[:, None], groups(H), 1)), (up, spread(up_s, H)), (down, spread(down_s, I)))
    return parts, lambda x: (x[:, at] * u * g)[:, to] * d


def tokens(M, H, fp32, seed):
    x = (fx.fp32_values if fp32 else fx.bf16_values)(M * H, seed).reshape(M, H)
    x[:, 0] = 1
    return x


@pytest.mark.parametrize("M,H,I,long", [(1, 2048, 1024, False), (5, 100, 33, False), (12, 256, 128, False), (40, 130, 70, False),
                                        (2, 64, 16384, False), (2800, 256, 512, True), (700, 2048, 1000, True)])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "bf16 weights"])
@pytest.mark.parametrize("group", [32, 128])
def test_gated_mlp_keeps_the_hidden_state(cuda_device, M, H, I, long, kind, group):
    from sb200 import _lib, group4
    fp32 = kind == "fp32"
    rows = 2 * M * H + 4 * M * (-(-I // 64) * 64) + 1024
    assert (_lib.load().sb_group4_gated_mlp_workspace_bytes(_lib.SB_BF16, M, H, I) > rows + 8 * H * I) is long
    parts, want = swiglu(H, I, M, group, fp32, kind == "bf16 weights")
    x = tokens(M, H, fp32, M)
    y = group4.gated_mlp(dev(x, cuda_device, torch.float32 if fp32 else torch.bfloat16),
                         *(matrix(c, s, group, cuda_device) for c, s in parts), out_dtype=torch.float32)
    same(y, want(x))


@pytest.mark.parametrize("B,k", [(1, 2), (2, 1), (5, 3), (40, 2), (200, 1)])
@pytest.mark.parametrize("H,I", [(256, 128), (130, 70), (2048, 96)])
@pytest.mark.parametrize("weights", ["ternary", "group4"])
@pytest.mark.parametrize("fp32", [False, True])
def test_few_token_layer_keeps_the_hidden_state(cuda_device, B, k, H, I, weights, fp32):
    """Routed to k experts, all but one of them with weight 0: that one's output, bit for bit, through
    the one-kernel sum and through the products by expert."""
    from sb200 import group4, ternary
    E, group = 4, 64
    layers = [swiglu(H, I, 10 * e, group, fp32, False) for e in range(E)]
    if weights == "group4":
        experts = group4.Group4Experts.pack(*({"codes": torch.from_numpy(np.stack([p[i][0] for p, _ in layers])).to(cuda_device),
                                               "scales": torch.from_numpy(np.stack([p[i][1] for p, _ in layers])).to(cuda_device)}
                                              for i in range(3)), group=group)
    else:
        t = [torch.from_numpy(np.stack([(p[i][0].astype(np.int8) - 8) for p, _ in layers])).to(cuda_device) for i in range(3)]
        s = [torch.from_numpy(np.stack([p[i][1][:, 0] for p, _ in layers])).float().to(cuda_device) for i in range(3)]
        experts = ternary.TernaryExperts.from_tensors(*t, *s)
    x = tokens(B, H, fp32, B + 1)
    rng = np.random.default_rng(B)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(B)]).astype(np.int32)
    w = np.zeros((B, k), np.float32)
    w[:, -1] = 1
    y = experts.forward_few(dev(x, cuda_device, torch.float32 if fp32 else torch.bfloat16),
                            torch.from_numpy(ids).to(cuda_device), torch.from_numpy(w).to(cuda_device))
    outs = np.stack([f(x) for _, f in layers])
    same(y, outs[ids[:, -1], np.arange(B)])
