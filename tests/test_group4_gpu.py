"""4-bit group weights on the GPU against the float64 restatement (needs a B200).

Tolerances come from ``oracle.group4``: a bound of fp32 sums for these very inputs,
plus half a step of the output type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import group4 as og

pytestmark = pytest.mark.gpu


def make(N, K, group, zeros, device, seed=0, raw=False):
    """A matrix of random codes and scales: (Group4Matrix, float64 values[, what it was packed from])."""
    from sb200 import group4
    rng = np.random.default_rng(seed)
    G = -(-K // group)
    codes = rng.integers(0, 16, (N, K)).astype(np.uint8)
    scales = og.bf16(rng.uniform(0.5, 1.5, (N, G)) / np.sqrt(K) / 4)
    z = rng.integers(0, 16, (N, G)).astype(np.uint8) if zeros else None
    parts = (torch.from_numpy(codes).to(device), torch.from_numpy(scales).to(device).bfloat16(),
             None if z is None else torch.from_numpy(z).to(device))
    m = group4.Group4Matrix.pack(*parts, group)
    return (m, og.values(codes, scales, z, group)) + ((parts,) if raw else ())


def acts(M, K, dtype, device, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(M, K, generator=g).to(dtype).to(device)


def close(y, ref, bound, what=""):
    got = y.double().cpu().numpy()
    b = og.rounded(ref, bound, str(y.dtype).replace("torch.", ""))
    worst = np.max(np.abs(got - ref) / np.maximum(b, 1e-300))
    print(f"{what}: {worst:.3f} of the bound")
    assert got.shape == ref.shape and worst <= 1.0, (what, worst)


# ---------------------------------------------------------------------------
# layout and quantiser
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("N,K", [(1, 1), (3, 8), (17, 127), (5, 128), (9, 129), (33, 1000)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_pack_and_dequantize(cuda_device, N, K, group, zeros):
    from sb200 import group4
    m, v, raw = make(N, K, group, zeros, cuda_device, seed=N + K, raw=True)
    np.testing.assert_array_equal(m.dequantize().double().cpu().numpy(), v)
    np.testing.assert_array_equal(m.dequantize(torch.bfloat16).double().cpu().numpy(), og.bf16(v))
    assert m.memory_bytes() == -(-N // 16) * -(-K // 128) * (1024 + 128 // group * (48 if zeros else 32))
    several = group4.Group4Matrix.pack(*(None if t is None else t.cpu().to(cuda_device).expand(3, *t.shape) for t in raw), group)
    np.testing.assert_array_equal(several.dequantize().double().cpu().numpy(), np.concatenate([v] * 3))
    np.testing.assert_array_equal(several.scales.cpu().float().numpy(), np.concatenate([raw[1].float().cpu().numpy()] * 3))


@pytest.mark.parametrize("N,K", [(1, 1), (2, 31), (7, 33), (16, 128), (5, 500), (64, 1029)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_equals_its_definition(cuda_device, N, K, group, symmetric, dtype):
    from sb200 import group4
    w = acts(N, K, dtype, cuda_device, seed=K)
    w[0] = 0                                  # a row of zeros: scale 0
    if N > 2:
        w[1] = w[1].abs() + 1                 # one sign only
        w[2] = torch.round(w[2] * 4) / 4      # quotients on ties
    m, vals = group4.quantize(w, group, symmetric, values=True)
    codes, scales, zeros = og.quantize(w.double().cpu().numpy(), group, symmetric)
    np.testing.assert_array_equal(m.scales.double().cpu().numpy(), scales)
    if not symmetric:
        np.testing.assert_array_equal(m.zeros.cpu().numpy(), zeros)
    ref = og.values(codes, scales, zeros, group)
    np.testing.assert_array_equal(vals.double().cpu().numpy(), ref)
    np.testing.assert_array_equal(m.dequantize().double().cpu().numpy(), ref)


def test_quantize_ties_that_fp32_division_hides(cuda_device):
    """Quotients that lie within fp32's rounding of a tie: w = (q + 1/2) s times 1 +- 2^-24."""
    from sb200 import group4
    s = np.float32(1.0 + 2.0 ** -7)                       # a bf16 scale: absmax = 7 s
    q = np.arange(-6, 7, dtype=np.float32) + np.float32(0.5)
    tie = (q * s).astype(np.float32)
    near = np.stack([tie, np.nextafter(tie, np.float32(np.inf)), np.nextafter(tie, np.float32(-np.inf))])
    w = np.zeros((3, 32), np.float32)
    w[:, 0] = np.float32(7) * s
    w[:, 1:14] = near
    m, vals = group4.quantize(torch.from_numpy(w).to(cuda_device), 32, True, values=True)
    codes, scales, zeros = og.quantize(w, 32, True)
    np.testing.assert_array_equal(vals.double().cpu().numpy(), og.values(codes, scales, zeros, 32))
    assert float(m.scales[0, 0]) == s


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize_non_finite_groups(cuda_device, symmetric):
    from sb200 import group4
    w = acts(4, 256, torch.float32, cuda_device, seed=3)
    w[0, 5], w[1, 70], w[2, 200] = float("nan"), float("inf"), -float("inf")
    m, vals = group4.quantize(w, 64, symmetric, values=True)
    bad = torch.zeros(4, 4, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 3] = True
    assert torch.equal(m.scales.isnan().cpu(), bad)
    assert torch.equal(vals.isnan().cpu(), bad.repeat_interleave(64, 1))


def test_quantize_extremes(cuda_device):
    """The largest and smallest fp32 weights; an asymmetric span past fp32 is a NaN scale."""
    from sb200 import group4
    big = torch.finfo(torch.float32).max
    w = torch.tensor([[big, -big] * 16, [1e-45, -1e-45] * 16, [1e-38, 2e-38] * 16], device=cuda_device)
    m, vals = group4.quantize(w, 32, True, values=True)
    codes, scales, zeros = og.quantize(w.double().cpu().numpy(), 32, True)
    np.testing.assert_array_equal(m.scales.double().cpu().numpy(), scales)
    # products past fp32's range or below its smallest step are rounded there
    np.testing.assert_array_equal(vals.cpu().numpy(), og.values(codes, scales, zeros, 32).astype(np.float32))
    m = group4.quantize(w, 32, False)
    assert m.scales[0].isnan().all() and m.scales[1:].isfinite().all()


def test_quantize_strided_rows(cuda_device):
    from sb200 import group4
    base = acts(40, 400, torch.float32, cuda_device, seed=5)
    for w in (base[:, 3:203], base[::2, :256], base.t()[:128]):
        a, va = group4.quantize(w, 64, False, values=True)
        b, vb = group4.quantize(w.contiguous(), 64, False, values=True)
        assert torch.equal(a.data, b.data) and torch.equal(va, vb) and torch.equal(a.scales, b.scales)


def test_pack_reports_codes_past_15(cuda_device):
    from sb200 import _lib, group4
    codes = torch.full((2, 128), 3, dtype=torch.uint8, device=cuda_device)
    one = torch.ones(2, 1, device=cuda_device)
    codes[1, 7] = 19
    m = group4.Group4Matrix.pack(codes, one)
    torch.cuda.synchronize()
    assert _lib.load().sb_device_status(0) == -1
    assert float(m.dequantize()[1, 7]) == 3 - 8
    group4.Group4Matrix.pack(codes & 15, one, torch.tensor([[3], [16]], dtype=torch.uint8, device=cuda_device))
    torch.cuda.synchronize()
    assert _lib.load().sb_device_status(0) == -1


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------

SHAPES = [(1, 16384, 20), (9, 16383, 33), (319, 72, 48), (320, 72, 48), (1, 8, 1), (1, 2048, 2048), (2, 64, 16), (7, 1000, 777), (8, 129, 33), (9, 128, 100), (16, 512, 48),
          (17, 264, 31), (33, 96, 130), (70, 2040, 65), (300, 256, 512), (513, 130, 260)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group,zeros,bias", [(32, True, True), (128, False, False), (64, True, False)])
def test_linear(cuda_device, M, K, N, dtype, group, zeros, bias):
    from sb200 import group4
    w, v = make(N, K, group, zeros, cuda_device, seed=M + N)
    x = acts(M, K, dtype, cuda_device, seed=K)
    b = torch.randn(N, generator=torch.Generator().manual_seed(2)).to(cuda_device) if bias else None
    fp32 = dtype == torch.float32
    xd = x.double().cpu().numpy()
    ref, bound = og.product(xd, v, np.abs(xd) * (2.0 ** -24 if fp32 else 0), 3 if fp32 else 2)
    if bias:
        bd = b.double().cpu().numpy()
        ref, bound = ref + bd, bound + og.STEP * (np.abs(ref) + np.abs(bd))
    y = group4.linear(x, w, b)
    assert y.dtype == dtype
    close(y, ref, bound, "linear")
    close(group4.linear(x, w, b, out_dtype=torch.float32), ref, bound, "linear fp32 out")


@pytest.mark.parametrize("M,H,I", [(1, 2048, 1024), (1, 72, 40), (3, 100, 33), (9, 256, 128), (40, 130, 70),
                                   (300, 256, 96), (600, 128, 200), (2, 16384, 17), (3, 33, 16384), (511, 72, 40), (512, 72, 41)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group,zeros", [(32, False), (128, True)])
def test_gated_mlp(cuda_device, M, H, I, dtype, group, zeros):
    from sb200 import group4
    ms = [make(n, k, group, zeros, cuda_device, seed=i) for i, (n, k) in enumerate([(I, H), (I, H), (H, I)])]
    x = acts(M, H, dtype, cuda_device, seed=M)
    y = group4.gated_mlp(x, *(m for m, _ in ms))
    ref, bound = og.gated_mlp(x.double().cpu().numpy(), *(v for _, v in ms), fp32=dtype == torch.float32)
    assert y.dtype == dtype
    close(y, ref, bound, "gated_mlp")
    close(group4.gated_mlp(x, *(m for m, _ in ms), out_dtype=torch.float32), ref, bound, "gated_mlp fp32 out")


def test_linear_rows_strides_and_shapes(cuda_device):
    """Leading dimensions, row strides, unaligned and transposed activations, out=, no tokens."""
    from sb200 import group4
    w, v = make(50, 128, 64, True, cuda_device)
    base = acts(12, 400, torch.bfloat16, cuda_device, seed=9)
    for x in (base[:, :128], base[:, 1:129], base[::3, 8:136], base[:, :384].reshape(12, 3, 128), base[0, :128],
              acts(128, 12, torch.bfloat16, cuda_device, seed=4).t(), base[:1, :128].expand(5, 128)):
        y = group4.linear(x, w)
        assert y.shape == (*x.shape[:-1], 50)
        ref, bound = og.product(x.reshape(-1, 128).double().cpu().numpy(), v)
        close(y.reshape(-1, 50), ref, bound, str(tuple(x.stride())))
    out = torch.empty(12, 50, device=cuda_device)
    assert group4.linear(base[:, :128], w, out=out) is out
    assert torch.equal(out, group4.linear(base[:, :128], w, out_dtype=torch.float32))
    half = acts(12, 50, torch.bfloat16, cuda_device)
    square = make(50, 50, 64, False, cuda_device)[0]
    for bad in (half, base[:, :50]):
        with pytest.raises(RuntimeError, match="overlaps|contiguous"):
            group4.linear(bad, square, out=bad)
    with pytest.raises(RuntimeError, match="gradient"):
        group4.linear(base[:, :128].clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="do not end in"):
        group4.linear(base[:, :127], w)
    with pytest.raises(RuntimeError, match="dtype"):
        group4.linear(base[:, :128].half(), w)
    with pytest.raises(RuntimeError, match="one matrix"):
        group4.linear(base[:, :128], group4.quantize(torch.randn(2, 50, 128, device=cuda_device)))
    with pytest.raises(RuntimeError, match="bias"):
        group4.linear(base[:, :128], w, torch.zeros(49, device=cuda_device))
    assert group4.linear(base[:0, :128], w).shape == (0, 50)
    assert group4.gated_mlp(base[:0, :128], w, w, make(128, 50, 64, True, cuda_device)[0]).shape == (0, 128)


def test_rows_do_not_depend_on_their_neighbours(cuda_device):
    """A non-finite token stays in its own row; the others keep their bits."""
    from sb200 import group4
    w, _ = make(64, 256, 32, True, cuda_device)
    for dtype in (torch.bfloat16, torch.float32):
        for M in (5, 20, 200, 600):
            x = acts(M, 256, dtype, cuda_device, seed=M)
            clean = group4.linear(x, w)
            x[3, 17], x[4, 0] = float("nan"), float("inf")
            y = group4.linear(x, w)
            keep = torch.ones(M, dtype=torch.bool, device=cuda_device)
            keep[3] = keep[4] = False
            assert torch.equal(y[keep], clean[keep]) and not y[3:5].isfinite().any()


def test_linear_magnitudes(cuda_device):
    """Activations near both ends of bf16 and fp32 keep their relative accuracy."""
    from sb200 import group4
    w, v = make(40, 256, 128, False, cuda_device)
    for dtype in (torch.bfloat16, torch.float32):
        for scale in (2.0 ** 100, 2.0 ** -60):
            x = acts(6, 256, dtype, cuda_device, seed=8) * scale
            fp32 = dtype == torch.float32
            xd = x.double().cpu().numpy()
            ref, bound = og.product(xd, v, np.abs(xd) * (2.0 ** -24 if fp32 else 0), 3 if fp32 else 2)
            close(group4.linear(x, w, out_dtype=torch.float32), ref, bound, f"x{scale:g}")


def test_streams_and_graph(cuda_device):
    """On a side stream, captured, and replayed on new values; two graphs do not share state."""
    from sb200 import group4
    ms = [make(n, k, 64, True, cuda_device, seed=i)[0] for i, (n, k) in enumerate([(96, 200), (96, 200), (200, 96)])]
    x1, x2 = (acts(m, 200, torch.float32, cuda_device, seed=m) for m in (4, 30))
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        e1, e2 = group4.gated_mlp(x1, *ms), group4.gated_mlp(x2, *ms)
    side.synchronize()
    assert torch.equal(e1, group4.gated_mlp(x1, *ms))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1, stream=side):
        y1 = group4.gated_mlp(x1, *ms)
    with torch.cuda.graph(g2, stream=side):
        y2 = group4.gated_mlp(x2, *ms)
    other = torch.cuda.Stream(cuda_device)
    torch.cuda.synchronize()
    for _ in range(3):
        g1.replay()
        with torch.cuda.stream(other):
            g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(y1, e1) and torch.equal(y2, e2)
    x1.copy_(x2[:4])
    g1.replay()
    torch.cuda.synchronize()
    assert torch.equal(y1, group4.gated_mlp(x1, *ms))


def test_results_repeat(cuda_device):
    from sb200 import group4
    w, _ = make(333, 1000, 32, True, cuda_device)
    for M in (1, 12, 700):
        x = acts(M, 1000, torch.bfloat16, cuda_device, seed=M)
        y = group4.linear(x, w)
        for _ in range(3):
            assert torch.equal(y, group4.linear(x, w))


# ---------------------------------------------------------------------------
# long prompts
# ---------------------------------------------------------------------------

def _written_out(M, K, N):
    """Whether a bf16 product of these sizes has its weights written out (its workspace tells)."""
    from sb200 import _lib
    return _lib.load().sb_group4_linear_workspace_bytes(_lib.SB_BF16, M, K, N) > 2 * M * (-(-K // 8) * 8) + 255


@pytest.mark.parametrize("M,K,N,long", [(1072, 130, 1024, False), (1073, 130, 1024, True), (1300, 72, 1001, True),
                                        (200, 8184, 4100, True), (120, 8192, 8001, False), (125, 8192, 8001, True)])
@pytest.mark.parametrize("group,zeros", [(32, True), (128, False)])
def test_linear_of_a_long_prompt(cuda_device, M, K, N, long, group, zeros):
    from sb200 import group4
    assert _written_out(M, K, N) is long
    w, v = make(N, K, group, zeros, cuda_device, seed=M + N)
    x = acts(M, K, torch.bfloat16, cuda_device, seed=K)
    b = torch.randn(N, generator=torch.Generator().manual_seed(2)).to(cuda_device)
    ref, bound = og.product(x.double().cpu().numpy(), v, 0, 2)
    bd = b.double().cpu().numpy()
    ref, bound = ref + bd, bound + og.STEP * (np.abs(ref) + np.abs(bd))
    y = group4.linear(x, w, b)
    close(y, ref, bound, "linear")
    close(group4.linear(x, w, b, out_dtype=torch.float32), ref, bound, "linear fp32 out")
    wide = torch.empty(M, K + 9, dtype=torch.bfloat16, device=cuda_device)  # rows that cannot be loaded 16 bytes at a time
    wide[:, 1:K + 1] = x
    assert torch.equal(group4.linear(wide[:, 1:K + 1], w, b), y)


@pytest.mark.parametrize("M,H,I,group,zeros", [(2800, 256, 512, 32, True), (700, 2048, 1000, 64, False), (3000, 250, 500, 128, True),
                                               (200, 4096, 8192, 128, False)])
def test_gated_mlp_of_a_long_prompt(cuda_device, M, H, I, group, zeros):
    from sb200 import _lib, group4
    rows = 2 * M * H + 4 * M * (-(-I // 64) * 64) + 1024  # the tokens and two planes of hidden rows
    assert _lib.load().sb_group4_gated_mlp_workspace_bytes(_lib.SB_BF16, M, H, I) > rows + 8 * H * I  # and the weights' terms
    ms = [make(n, k, group, zeros, cuda_device, seed=i) for i, (n, k) in enumerate([(I, H), (I, H), (H, I)])]
    x = acts(M, H, torch.bfloat16, cuda_device, seed=M)
    ref, bound = og.gated_mlp(x.double().cpu().numpy(), *(v for _, v in ms), fp32=False)
    close(group4.gated_mlp(x, *(m for m, _ in ms)), ref, bound, "gated_mlp")
    close(group4.gated_mlp(x, *(m for m, _ in ms), out_dtype=torch.float32), ref, bound, "gated_mlp fp32 out")


def test_gradients_are_refused(cuda_device):
    from sb200 import group4
    w = make(48, 128, 64, False, cuda_device)[0]
    x = acts(3, 128, torch.bfloat16, cuda_device)
    b = torch.zeros(48, device=cuda_device, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradient"):
        group4.linear(x, w, b)
    with torch.no_grad():
        assert torch.equal(group4.linear(x, w, b), group4.linear(x, w))
    ex = group4.Group4Experts.quantize(*(torch.randn(2, n, k, device=cuda_device) for n, k in ((32, 128), (32, 128), (128, 32))))
    ids = torch.zeros(3, 1, dtype=torch.int32, device=cuda_device)
    with pytest.raises(RuntimeError, match="gradient"):
        ex.forward_few(x, ids, torch.ones(3, 1, device=cuda_device, requires_grad=True))


@pytest.mark.parametrize("M,K,N", [(5000, 72, 16), (4099, 40, 33), (2500, 136, 100)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_tokens_of_a_narrow_matrix(cuda_device, M, K, N, dtype):
    """Far more groups of tokens than blocks, a unit or a few to each."""
    from sb200 import group4
    w, v = make(N, K, 32, True, cuda_device, seed=N)
    x = acts(M, K, dtype, cuda_device, seed=M)
    fp32 = dtype == torch.float32
    xd = x.double().cpu().numpy()
    ref, bound = og.product(xd, v, np.abs(xd) * (2.0 ** -24 if fp32 else 0), 3 if fp32 else 2)
    close(group4.linear(x, w), ref, bound, "linear")


@pytest.mark.parametrize("group,zeros", [(32, True), (128, False)])
def test_data_inside_a_larger_buffer(cuda_device, group, zeros):
    """A matrix whose bytes are a slice of a checkpoint's: products, values, scales and zero points."""
    from sb200 import group4
    m, _ = make(50, 300, group, zeros, cuda_device)
    n = m.data.numel()
    buffer = torch.full((n + 4096,), 255, dtype=torch.uint8, device=cuda_device)
    buffer[1040:1040 + n] = m.data
    part = group4.Group4Matrix(buffer[1040:1040 + n], 50, 300, group, zeros)
    x = acts(5, 300, torch.bfloat16, cuda_device)
    assert torch.equal(group4.linear(x, part), group4.linear(x, m))
    assert torch.equal(part.dequantize(), m.dequantize()) and torch.equal(part.scales, m.scales)
    assert (part.zeros is None) if not zeros else torch.equal(part.zeros, m.zeros)
    with pytest.raises(RuntimeError, match="16-byte"):
        group4.Group4Matrix(buffer[1032:1032 + n], 50, 300, group, zeros)


@pytest.mark.parametrize("M", [1, 20, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_group_sums_of_large_activations(cuda_device, M, dtype):
    """A group's sum before its scale may be past fp32's range where the product is not:
    128 weights of 15 x 2^-20 on activations of 2^126."""
    from sb200 import group4
    K, N = 256, 1000
    w = group4.Group4Matrix.pack(torch.full((N, K), 15, dtype=torch.uint8, device=cuda_device),
                                 torch.full((N, 2), 2.0 ** -20, device=cuda_device),
                                 torch.zeros(N, 2, dtype=torch.uint8, device=cuda_device))
    x = torch.full((M, K), 2.0 ** 126, dtype=dtype, device=cuda_device)
    y = group4.linear(x, w, out_dtype=torch.float32)
    assert (y == 15 * 2.0 ** 114).all()                    # every partial sum is a whole multiple of 2^106 below 2^118: exact
    experts = group4.Group4Experts.pack(*({"codes": torch.full((1, n, k), 9, dtype=torch.uint8, device=cuda_device),
                                           "scales": torch.full((1, n, -(-k // 128)), s, device=cuda_device)}
                                          for n, k, s in ((128, K, 2.0 ** -100), (128, K, 2.0 ** -30), (K, 128, 2.0 ** -20))))
    ids = torch.zeros(M, 1, dtype=torch.int32, device=cuda_device)
    y = experts.forward_few(x * 2.0 ** -6, ids, torch.ones(M, 1, device=cuda_device))
    # gate 2^28, and silu of it the same; up 2^98; 128 hidden values of 2^126 at 2^-20
    assert (y == 2.0 ** 113).all()


@pytest.mark.parametrize("M", [2, 20])
def test_largest_and_infinite_fp32_values(cuda_device, M):
    """fp32 values that bf16 rounds to infinity stay what they are, and an infinity stays one:
    activations, and the hidden state of the gated MLP."""
    from sb200 import group4
    K, big = 128, torch.finfo(torch.float32).max
    codes = torch.full((3, K), 8, dtype=torch.uint8, device=cuda_device)
    codes[0, :], codes[1, 5], codes[2, 5:7] = 9, 9, 7     # row 0 meets every value, rows 1 and 2 the fifth (and sixth)
    w = group4.Group4Matrix.pack(codes, torch.full((3, 1), 2.0 ** -10, device=cuda_device))
    x = torch.zeros(M, K, device=cuda_device)
    for value in (big, -big, 3.3962e38, -3.4e38):
        x[:, 5] = value
        # one product, all planes of it: exact
        want = torch.tensor([1.0, 1.0, -1.0], dtype=torch.float64) * x[0, 5].item() * 2.0 ** -10
        assert torch.equal(group4.linear(x, w).double().cpu(), want.expand(M, 3))
    x[:, 5] = -torch.inf
    y = group4.linear(x, w)
    assert (y[:, 1] == -torch.inf).all() and (y[:, 2] == torch.inf).all()
    # silu(g) u = g u where exp(-g) is lost beside 1
    scale = lambda s, n: torch.tensor([[s]], device=cuda_device).expand(n, 1)  # noqa: E731
    gate, up = (group4.Group4Matrix.pack(codes[1:2].expand(8, K), scale(s, 8)) for s in (1.0, 2.0 ** -64))
    down = group4.Group4Matrix.pack(torch.full((K, 8), 9, dtype=torch.uint8, device=cuda_device), scale(2.0 ** -10, K))
    x.zero_()
    x[:, 5] = 2.0 ** 96 * (2.0 - 2.0 ** -23)              # h = (2 - 2^-23)^2 2^128, past fp32
    assert (group4.gated_mlp(x, gate, up, down) == torch.inf).all()
    x[:, 5] = 2.0 ** 96 * (1.0 - 2.0 ** -12)
    h = (1.0 - 2.0 ** -12) ** 2 * 2.0 ** 128              # 2^-24 from a whole fp32, and past bf16's largest
    assert 3.397e38 < h < big
    # eight equal terms of 2^-10 h: sums and the planes' additions are off by at most 2^-20 together
    y = group4.gated_mlp(x, gate, up, down).double().cpu()
    assert ((y / (8 * h * 2.0 ** -10) - 1).abs() < 2.0 ** -20).all()


def _term_order_weights(N, K, cuda_device):
    """Weights of 15 x 129/128 = 15.1171875, in two bf16 terms 15.125 and -2^-7."""
    from sb200 import group4
    codes = torch.full((N, K), 15, dtype=torch.uint8, device=cuda_device)
    scales = torch.full((N, -(-K // 128)), 129 / 128, device=cuda_device)
    return group4.Group4Matrix.pack(codes, scales, torch.zeros(N, -(-K // 128), dtype=torch.uint8, device=cuda_device))


def test_long_prompt_keeps_the_small_terms(cuda_device):
    """The weights' low terms of a long prompt are added up before the large sum that they would
    be truncated in: one activation of 2^18 beside 2047 ones.  The low terms' sum, a multiple of
    2^-7 below 2^12, the high terms', a multiple of 2^-3 below 2^15 before the 2^18, and the
    exact result's rounding: one step of 2^-23 for that, one for truncating it."""
    from sb200 import group4
    M, K, N = 1200, 2048, 1001
    assert _written_out(M, K, N)
    w = _term_order_weights(N, K, cuda_device)
    x = torch.ones(M, K, dtype=torch.bfloat16, device=cuda_device)
    x[:, -1] = 2.0 ** 18
    want = (15 * 129 / 128) * (K - 1 + 2.0 ** 18)
    y = group4.linear(x, w, out_dtype=torch.float32).double()
    assert ((y / want - 1).abs() <= 2 * 2.0 ** -23).all()


def test_long_mlp_keeps_the_small_terms(cuda_device):
    """The same of the gated MLP: its hidden values are 1 and, last, 2^18 (silu(32) = 32 in fp32),
    and the tokens' low terms of the gate and up products are exact."""
    from sb200 import _lib, group4
    M, H, I = 1500, 512, 2048
    rows = 2 * M * H + 4 * M * I + 1024
    assert _lib.load().sb_group4_gated_mlp_workspace_bytes(_lib.SB_BF16, M, H, I) > rows + 8 * H * I
    codes = torch.full((I, H), 8, dtype=torch.uint8, device=cuda_device)
    codes[:, 0] = 9
    scales = torch.full((I, H // 128), 32.0, device=cuda_device)
    ups = torch.full((I, H // 128), 2.0 ** -5, device=cuda_device)
    ups[-1] = 2.0 ** 13
    gate, up = group4.Group4Matrix.pack(codes, scales), group4.Group4Matrix.pack(codes, ups)
    x = torch.zeros(M, H, dtype=torch.bfloat16, device=cuda_device)
    x[:, 0] = 1
    want = (15 * 129 / 128) * (I - 1 + 2.0 ** 18)
    y = group4.gated_mlp(x, gate, up, _term_order_weights(H, I, cuda_device), out_dtype=torch.float32).double()
    assert ((y / want - 1).abs() <= 2 * 2.0 ** -23).all()


def test_out_that_overlaps_the_bias_is_refused(cuda_device):
    from sb200 import group4
    w = make(48, 128, 64, False, cuda_device)[0]
    x = acts(3, 128, torch.bfloat16, cuda_device)
    buffer = torch.zeros(4, 48, device=cuda_device)
    with pytest.raises(RuntimeError, match="overlaps the bias"):
        group4.linear(x, w, buffer[1], out=buffer[:3])
    y = group4.linear(x, w, buffer[3], out=buffer[:3])
    assert torch.equal(y, group4.linear(x, w, out_dtype=torch.float32))
