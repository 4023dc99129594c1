"""The MoE layer of the hot path: BVH router top-k -> grouped ternary SwiGLU.

``BVHMoELayer.forward(x)`` = router top-k (``BVHRouter.forward_topk``) followed by
``sum_j w[t,j] * expert_{ids[t,j]}(x[t])`` over ternary experts, i.e. the
composition the reference runs as ``BVHGateWrapper`` + the Python dispatch loop
of ``OLMoELayer.forward_topk`` (python/olmoe_extract.py:126-157) over
``CUDATernaryExpertModule`` experts (python/ternary_expert_ext_bridge.py:75-175).
Everything runs on the device: no host round trip between routing and experts.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import group4
from .ternary import TernaryExperts


class BVHMoELayer:
    def __init__(self, router, experts, top_k: int = 8, select: str = "soft",
                 device: Optional[torch.device] = None, few_tokens: int = 0):
        """router: a ``bvh_router.BVHRouter`` (on ``device``); experts: a
        ``TernaryExperts``, a ``group4.Group4Experts`` or a sequence of expert
        containers.  Batches of up to ``few_tokens`` tokens run the ternary experts
        through ``forward_few`` (for decoding: a fraction of the time up to some 150
        tokens, another order of the sums); 4-bit experts always do, in calls of
        ``group4.max_tokens(top_k)`` tokens."""
        self.router = router
        self.device = torch.device(device) if device is not None else router.to_3d.weight.device
        ready = isinstance(experts, (TernaryExperts, group4.Group4Experts))
        self.experts = experts if ready else TernaryExperts(experts, self.device)
        self.top_k = int(top_k)
        self.select = select
        self.few_tokens = int(few_tokens)

    def route(self, x: torch.Tensor):
        return self.router.forward_topk(x, k=self.top_k, select=self.select)

    def forward(self, x: torch.Tensor, out_dtype=None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        ids, w = self.route(x)
        return self._run(x, ids, w, out_dtype or x.dtype, out)

    def _run(self, x, ids, w, out_dtype, out=None) -> torch.Tensor:
        few = 0 < ids.shape[0] <= self.few_tokens
        f = self.experts.forward_few if few else self.experts.forward
        return f(x, ids, w, out_dtype=out_dtype, out=out)

    __call__ = forward

    def forward_topk(self, hidden_states: torch.Tensor, topk_probs: torch.Tensor,
                     topk_ids: torch.Tensor) -> torch.Tensor:
        """Same signature as OLMoELayer.forward_topk (olmoe_extract.py:126-157)."""
        return self._run(hidden_states, topk_ids, topk_probs, hidden_states.dtype)


class FewTokenMoE:
    """A whole MoE layer for decoding batches: dense gate, softmax, top-k, SwiGLU
    experts and their weighted sum, in three to five kernels (six for fp32 rows).

    ``gate_weight`` [E, H] (fp32 or bf16, an ``nn.Linear`` weight, read as it is at
    each call) scores the experts; a token's weights are its ``top_k`` largest softmax probabilities, in
    descending order, divided by their sum with ``norm_topk`` (the gate of
    OlmoeTopKRouter and of the hybrid gate's dense part, without rounding the
    logits to the hidden dtype).  ``experts``: ``TernaryExperts`` or
    ``group4.Group4Experts``.  Any batch runs, cut into calls of
    ``group4.max_tokens(top_k)`` tokens.  For ternary experts the grouped layer
    (``BVHMoELayer``, ``TernaryExperts.forward``) is the faster one past some 150 tokens
    (64 experts of 2048 x 1024, top 8: 123 us here and 139 there at 128, 166 and 140 at
    192); 4-bit experts have no other form.
    """

    def __init__(self, experts, gate_weight: torch.Tensor, top_k: int = 8, norm_topk: bool = False):
        E, H = experts.E, experts.H
        if tuple(gate_weight.shape) != (E, H):
            raise RuntimeError(f"gate_weight of shape {tuple(gate_weight.shape)} must be [{E}, {H}]")
        if gate_weight.device != experts.gate.device:
            raise RuntimeError(f"gate_weight is on {gate_weight.device}, the experts are on {experts.gate.device}")
        if not 1 <= int(top_k) <= min(E, 32):
            raise RuntimeError(f"top_k {top_k} is not in 1..{min(E, 32)}")
        if gate_weight.dtype not in (torch.float32, torch.bfloat16):
            raise RuntimeError(f"gate dtype {gate_weight.dtype} must be float32 or bfloat16")
        group4.check_experts(E, H, experts.I)
        self.experts = experts
        self.gate_weight = gate_weight
        self.top_k = int(top_k)
        self.norm_topk = bool(norm_topk)

    def __call__(self, x: torch.Tensor, out_dtype=None, out: Optional[torch.Tensor] = None, routing: bool = False):
        """The layer's output, of x's shape and (unless ``out_dtype`` or ``out`` says
        otherwise) dtype; with ``routing`` (output, ids int32 [tokens, k], weights fp32)."""
        y, ids, w = group4.few_moe(self.experts, x, None, None, self.gate_weight, self.top_k, self.norm_topk,
                                   out_dtype=out_dtype, out=out, routing=routing)
        return (y, ids, w) if routing else y


class GraphedLayer:
    """A layer replayed from CUDA graphs: the first call with a given
    (input, output) buffer pair runs the layer twice to warm every cached
    workspace and kernel attribute, then captures one forward into a graph;
    later calls with the same buffers replay it on the current stream (one
    launch instead of the layer's eight, no per-kernel launch gaps).

    Valid while the buffers, the batch shape and the layer's weights stay in
    place: a weight re-upload that moves device memory needs ``reset()``.
    Calls with new buffers capture another graph (up to ``max_graphs``).
    """

    def __init__(self, layer, max_graphs: int = 8):
        self.layer = layer
        self.max_graphs = int(max_graphs)
        self._graphs = {}

    def reset(self) -> None:
        self._graphs.clear()

    def _key(self, x: torch.Tensor, out: torch.Tensor):
        return (x.data_ptr(), tuple(x.shape), x.dtype, out.data_ptr(), tuple(out.shape), out.dtype)

    def __call__(self, x: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
        key = self._key(x, out)
        g = self._graphs.get(key)
        if g is None:
            if len(self._graphs) >= self.max_graphs:
                self._graphs.pop(next(iter(self._graphs)))
            cur = torch.cuda.current_stream(x.device)
            side = torch.cuda.Stream(x.device)
            side.wait_stream(cur)
            with torch.cuda.stream(side):
                for _ in range(2):
                    self.layer(x, out=out)
            cur.wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                self.layer(x, out=out)
            cur.wait_stream(side)
            self._graphs[key] = g
        g.replay()
        return out


class HostPipeline:
    """Runs a stream of host-resident batches through a layer with the copies
    overlapped: while the layer computes batch i on the compute stream, batch
    i+1 is copied in on one copy stream and batch i-1's result copied out on
    another (two device buffers each way).  Every batch still makes its full
    host->device and device->host trip; only their timing overlaps.

    ``layer`` is any callable ``layer(x_dev, out=y_dev)`` on the device, such as
    ``BVHMoELayer``.  Host tensors should be pinned for the copies to be
    asynchronous.
    """

    def __init__(self, layer, batch: int, hidden: int, dtype=torch.bfloat16,
                 device: Optional[torch.device] = None, out_dtype=None):
        self.layer = layer
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.xin = [torch.empty(batch, hidden, dtype=dtype, device=self.device) for _ in range(2)]
        self.yout = [torch.empty(batch, hidden, dtype=out_dtype or dtype, device=self.device) for _ in range(2)]
        self.h2d = torch.cuda.Stream(self.device)
        self.d2h = torch.cuda.Stream(self.device)
        ev = lambda: [torch.cuda.Event() for _ in range(2)]
        self.in_ready, self.in_free, self.out_ready, self.out_free = ev(), ev(), ev(), ev()

    def run(self, inputs: Sequence[torch.Tensor], outputs: Sequence[torch.Tensor]) -> None:
        """outputs[i] <- layer(inputs[i]) for every i; returns when all copies are queued
        (synchronise the current stream, or wait on ``done_event``, to read them)."""
        compute = torch.cuda.current_stream(self.device)
        start = torch.cuda.Event()
        start.record(compute)
        self.h2d.wait_event(start)
        self.d2h.wait_event(start)
        for i, (xh, yh) in enumerate(zip(inputs, outputs)):
            b = i & 1
            with torch.cuda.stream(self.h2d):
                if i >= 2:
                    self.h2d.wait_event(self.in_free[b])   # compute of batch i-2 has read xin[b]
                self.xin[b].copy_(xh, non_blocking=True)
                self.in_ready[b].record(self.h2d)
            compute.wait_event(self.in_ready[b])
            if i >= 2:
                compute.wait_event(self.out_free[b])       # batch i-2's result has left yout[b]
            self.layer(self.xin[b], out=self.yout[b])
            self.in_free[b].record(compute)
            self.out_ready[b].record(compute)
            with torch.cuda.stream(self.d2h):
                self.d2h.wait_event(self.out_ready[b])
                yh.copy_(self.yout[b], non_blocking=True)
                self.out_free[b].record(self.d2h)
        # the caller's stream is done when the last copy out is
        last = (len(inputs) - 1) & 1 if len(inputs) else 0
        if len(inputs):
            compute.wait_event(self.out_free[last])
            if len(inputs) > 1:
                compute.wait_event(self.out_free[last ^ 1])
