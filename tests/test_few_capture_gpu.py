"""The few-token kernels in captured graphs behind copies, memsets and joined streams, and called by
several threads at once (needs a B200).  Their launches may begin before the kernel in front of them
has ended, which must hold behind anything else, too."""

from __future__ import annotations

import threading

import pytest
import torch

from test_group4_gpu import acts, make
from test_moe_few_gpu import make_experts

pytestmark = pytest.mark.gpu


def layers(cuda_device):
    """name -> (call(x), K) over one set of weights, fp32 and bf16, one and two kernels and more."""
    from sb200 import group4
    from sb200.moe import FewTokenMoE
    w = make(96, 200, 64, True, cuda_device)[0]
    ms = [make(n, k, 64, True, cuda_device, seed=i)[0] for i, (n, k) in enumerate([(96, 200), (96, 200), (200, 96)])]
    ex, _ = make_experts("group4", 8, 200, 48, cuda_device)
    gate = acts(8, 200, torch.float32, cuda_device, seed=77) / 14
    layer = FewTokenMoE(ex, gate, 3)
    return {"linear": lambda x: group4.linear(x, w), "mlp": lambda x: group4.gated_mlp(x, *ms), "layer": layer}


@pytest.mark.parametrize("name", ["linear", "mlp", "layer"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M", [1, 30])
def test_captured_behind_other_work(cuda_device, name, dtype, M):
    call = layers(cuda_device)[name]
    x1, x2 = (acts(M, 200, dtype, cuda_device, seed=s) for s in (1, 2))
    want1, want2, want0 = call(x1), call(x2), call(torch.zeros_like(x1))
    x, held = torch.empty_like(x1), torch.empty_like(x1)
    side, other = torch.cuda.Stream(cuda_device), torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        x.copy_(x1)                       # a copy in front of the call
        a = call(x)
        x.zero_()                         # and a memset
        b = call(x)
        other.wait_stream(side)           # two branches, joined in front of the call
        with torch.cuda.stream(other):
            held.copy_(x2)
            c = call(held)
        x.copy_(x1)
        d = call(x)
        side.wait_stream(other)
        e = call(held)
        held.copy_(x1)                    # what follows may not overtake the call
        x.copy_(x2)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for got, want in ((a, want1), (b, want0), (c, want2), (d, want1), (e, want2)):
        assert torch.equal(got, want)


def test_calls_of_several_threads(cuda_device):
    """Four threads, a stream each, one set of weights."""
    calls = layers(cuda_device)
    xs = [acts(M, 200, dtype, cuda_device, seed=M) for M in (1, 7, 20, 64) for dtype in (torch.bfloat16, torch.float32)]
    want = {name: [call(x) for x in xs] for name, call in calls.items()}
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream(cuda_device)
        with torch.cuda.stream(stream):
            for r in range(10):
                for name, call in calls.items():
                    got = [call(x) for x in xs]
                    stream.synchronize()
                    bad.extend((i, r, name, j) for j, (g, w) in enumerate(zip(got, want[name])) if not torch.equal(g, w))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad[:5]
