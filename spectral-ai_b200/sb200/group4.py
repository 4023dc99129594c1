"""Weights in 4-bit groups: quantiser, products and experts.

A matrix [N, K] is held as 4-bit codes with a bf16 scale (and, if asymmetric, a
zero point) for each row and group of 32, 64 or 128 along K:

    W[n, k] = scale[n, k // G] * (code[n, k] - zero[n, k // G])    (zero 8 if none)

``quantize`` makes such a matrix from weights, ``Group4Matrix.pack`` from codes
and scales that another quantiser chose; ``linear`` and ``gated_mlp`` are the
products of a layer's activations with them, from one token to a long prompt;
``Group4Experts`` holds a layer's experts and stands where
``sb200.ternary.TernaryExperts`` does, at 4 bits a weight instead of 2.

Everything runs on the device of its tensors and on its current stream, and can
be captured into a CUDA graph.  There is no backward.
"""

from __future__ import annotations

import contextlib
import ctypes as C
import functools
import math
from typing import Optional

import torch

from . import _lib

GROUPS = (32, 64, 128)
MAX_WIDTH, MAX_EXPERTS = 8192, 512  # H and I, and E, of the few-token layer


_NOWHERE = contextlib.nullcontext()
_CODES = {torch.float32: _lib.SB_F32, torch.bfloat16: _lib.SB_BF16}


def _on(device: torch.device):
    """The device's context, entered only where it is not the current one."""
    return _NOWHERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _workspace(nbytes: int, device) -> torch.Tensor:
    """A workspace of its own for every call: the caching allocator orders its
    reuse on the stream, and a captured graph keeps it in its own pool."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _code(dtype: torch.dtype, what: str) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise RuntimeError(f"{what} dtype {dtype} must be float32 or bfloat16")
    return code


def _check_cuda(t, what: str, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{what} must be a CUDA tensor (there is no CPU path)")
    if device is not None and t.device != device:
        raise RuntimeError(f"{what} is on {t.device}, the weights are on {device}")


def _no_grad(t: torch.Tensor, what: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} require a gradient and there is no backward; call this under torch.no_grad()")


def _rows(x: torch.Tensor, K: int, device: torch.device):
    """x [..., K] as rows with unit stride along K (copied only where it has another):
    (rows, their count, their stride)."""
    _check_cuda(x, "activations", device)
    shape = x.shape
    if not shape or shape[-1] != K:
        raise RuntimeError(f"activations of shape {tuple(shape)} do not end in {K}")
    _no_grad(x, "activations")
    if len(shape) != 2:
        x = x.reshape(-1, K)
    M = x.shape[0]
    ld, unit = x.stride()
    if (unit != 1 and K > 1) or (ld < K and M > 1):
        x, ld = x.contiguous(), K
    return x, M, max(ld, K)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory from one tensor's first to its last element meets the other's."""
    if a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr() or not a.numel() or not b.numel():
        return False
    end = lambda t: t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))  # noqa: E731
    return a.data_ptr() < end(b) and b.data_ptr() < end(a)


def _output(out, shape, dtype, device, **inputs) -> torch.Tensor:
    """``out``, checked, or a new tensor; ``inputs`` (by name) are read while it is written."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _check_cuda(out, "out", device)
    if tuple(out.shape) != tuple(shape) or not out.is_contiguous():
        raise RuntimeError(f"out must be contiguous of shape {tuple(shape)}, got {tuple(out.shape)}")
    for what, t in inputs.items():
        if t is not None and _overlap(out, t):
            raise RuntimeError(f"out overlaps the {what.replace('_', ' ')}, which are read while it is written")
    return out


class Group4Matrix:
    """``count`` matrices [N, K] in 4-bit groups on one device.  ``data`` (uint8) holds
    them in the library's block layout (include/spectral_b200.h); it is not replaced
    once the object is made."""

    def __init__(self, data: torch.Tensor, N: int, K: int, group: int, zeros: bool, count: int = 1):
        if group not in GROUPS:
            raise RuntimeError(f"group {group} must be one of {GROUPS}")
        _check_cuda(data, "data")
        self.N, self.K, self.group, self.count, self.has_zeros = int(N), int(K), int(group), int(count), bool(zeros)
        need = self.count * _matrix_bytes(self.K, self.N, self.group, self.has_zeros)
        if min(self.N, self.K, self.count) < 1 or data.dtype != torch.uint8 or not data.is_contiguous() \
                or data.numel() != need:
            raise RuntimeError(f"{self.count} matrices [{N}, {K}] in groups of {group} are {need} contiguous bytes, got "
                               f"{data.dtype} {tuple(data.shape)}")
        if data.data_ptr() % 16:
            raise RuntimeError("data must start on a 16-byte boundary")
        self.data, self.device = data, data.device
        self.desc = _lib.Group4(data.data_ptr(), self.K, self.N, self.count, self.group, int(self.has_zeros))
        self.ref = C.byref(self.desc)

    @classmethod
    def _empty(cls, shape, group: int, zeros: bool, device) -> "Group4Matrix":
        """Room for matrices of ``shape`` [..., N, K]."""
        if group not in GROUPS:
            raise RuntimeError(f"group {group} must be one of {GROUPS}")
        if len(shape) < 2 or min(shape) < 1:
            raise RuntimeError(f"weights of shape {tuple(shape)} must be [..., N, K] and not empty")
        count = math.prod(shape[:-2])
        N, K = shape[-2:]
        data = torch.empty(count * _matrix_bytes(K, N, group, zeros), dtype=torch.uint8, device=device)
        return cls(data, N, K, group, zeros, count)

    @classmethod
    def pack(cls, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
             group: int = 128) -> "Group4Matrix":
        """From codes uint8 [..., N, K] in 0..15 (leading dimensions count matrices), scales
        [..., N, ceil(K/group)] (kept as bf16) and zero points uint8 in 0..15 or None."""
        _check_cuda(codes, "codes")
        if codes.dtype != torch.uint8:
            raise RuntimeError(f"codes must be uint8, got {codes.dtype}")
        m = cls._empty(codes.shape, group, zeros is not None, codes.device)
        shape = (*codes.shape[:-1], -(-m.K // group))
        for t, what in ((scales, "scales"), (zeros, "zeros")):
            if t is not None:
                _check_cuda(t, what, codes.device)
                if tuple(t.shape) != shape:
                    raise RuntimeError(f"{what} of shape {tuple(t.shape)} must be {shape}")
        if zeros is not None and zeros.dtype != torch.uint8:
            raise RuntimeError(f"zeros must be uint8, got {zeros.dtype}")
        codes, scales = codes.contiguous(), scales.detach().to(torch.bfloat16).contiguous()
        zeros = None if zeros is None else zeros.contiguous()
        with _on(codes.device):
            _lib.check(_lib.load().sb_group4_pack(codes.data_ptr(), scales.data_ptr(), _ptr(zeros), m.ref,
                                                  _stream(codes.device)), "sb_group4_pack")
        return m

    def _rows(self, flat: torch.Tensor, block: int, offset: int) -> torch.Tensor:
        """Scales or zero points (``flat``: the data as their type, which may begin anywhere
        in its storage, ``block`` of it to a block, theirs from ``offset``) row-major:
        [count * N, groups], one copy."""
        tiles, chunks, per = (self.N + 15) // 16, (self.K + 127) // 128, 128 // self.group
        t = flat.as_strided((self.count, tiles, 2, 8, chunks, per), (tiles * chunks * block, chunks * block, 1, 2, block, 16),
                            flat.storage_offset() + offset)
        t = t.reshape(self.count, tiles * 16, chunks * per)[:, :self.N, :-(-self.K // self.group)]
        return t[0] if self.count == 1 else t.reshape(self.count * self.N, -1)

    @property
    def scales(self) -> torch.Tensor:
        """bf16 [count * N, ceil(K/group)], a copy."""
        per = 128 // self.group
        return self._rows(self.data.view(torch.bfloat16), 512 + (24 if self.has_zeros else 16) * per, 512)

    @property
    def zeros(self) -> Optional[torch.Tensor]:
        """uint8 [count * N, ceil(K/group)], a copy, or None."""
        per = 128 // self.group
        return self._rows(self.data, 1024 + 48 * per, 1024 + 32 * per) if self.has_zeros else None

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values [count * N, K], exact in fp32, rounded in bf16."""
        out = torch.empty(self.count * self.N, self.K, dtype=dtype, device=self.device)
        with _on(self.device):
            _lib.check(_lib.load().sb_group4_dequantize(self.ref, out.data_ptr(), _code(dtype, "value"),
                                                        _stream(self.device)), "sb_group4_dequantize")
        return out

    def memory_bytes(self) -> int:
        return self.data.numel()


def _matrix_bytes(K: int, N: int, group: int, zeros: bool) -> int:
    return int(_lib.load().sb_group4_matrix_bytes(K, N, group, int(zeros)))


def _stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)  # torch.cuda.current_stream's, without the object around it


def quantize(w: torch.Tensor, group: int = 128, symmetric: bool = True, values: bool = False):
    """Weights [..., N, K] (fp32 or bf16) -> ``Group4Matrix`` (leading dimensions count
    matrices).

    Symmetric: scale = absmax / 7 and codes around 8; else scale = (max - min) / 15
    with 0 in the range and a zero point.  Nearest codes, ties to even.  A group with
    a non-finite weight gets a NaN scale.  With ``values`` also returns what the codes
    stand for, fp32 [count * N, K]."""
    _check_cuda(w, "weights")
    code = _code(w.dtype, "weight")
    m = Group4Matrix._empty(w.shape, group, not symmetric, w.device)
    w = w.detach()
    w = w if w.dim() == 2 else w.reshape(-1, m.K)
    if (w.stride(1) != 1 and m.K > 1) or (w.stride(0) < m.K and w.shape[0] > 1):
        w = w.contiguous()
    vals = torch.empty(w.shape[0], m.K, dtype=torch.float32, device=w.device) if values else None
    with _on(w.device):
        _lib.check(_lib.load().sb_group4_quantize(w.data_ptr(), code, max(w.stride(0), m.K), m.ref, _ptr(vals),
                                                  _stream(w.device)), "sb_group4_quantize")
    return (m, vals) if values else m


@functools.lru_cache(maxsize=1024)
def _linear_bytes(xc: int, M: int, K: int, N: int) -> int:
    return int(_lib.load().sb_group4_linear_workspace_bytes(xc, M, K, N))


def linear(x: torch.Tensor, w: Group4Matrix, bias: Optional[torch.Tensor] = None, out_dtype=None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[..., N] = x W^T (+ bias), in x's dtype unless ``out_dtype`` (or ``out``, which overlaps no
    input) says fp32 or bf16."""
    lib, dev = _lib.load(), w.device
    x2, M, ldx = _rows(x, w.K, dev)
    if bias is not None:
        _check_cuda(bias, "bias", dev)
        if bias.shape != (w.N,):
            raise RuntimeError(f"bias of shape {tuple(bias.shape)} must be [{w.N}]")
        _no_grad(bias, "the bias's values")
        if bias.dtype != torch.float32 or not bias.is_contiguous():
            bias = bias.detach().to(torch.float32).contiguous()
    y = _output(out, (*x.shape[:-1], w.N), out_dtype or x.dtype, dev, activations=x2, bias_values=bias)
    xc, xp, ws, need = _code(x2.dtype, "activation"), x2.data_ptr(), None, 0
    if xc != _lib.SB_BF16 or w.K % 8 or ldx % 8 or xp % 16 or _linear_bytes(xc, M, w.K, w.N) > 2 * M * w.K + 255:
        need = _linear_bytes(xc, M, w.K, w.N)
        ws = _workspace(need, dev)  # (else it would hold no more than the rows, which are read in place)
    with _on(dev):
        rc = lib.sb_group4_linear(xp, xc, ldx, M, w.ref, _ptr(bias), y.data_ptr(), _code(y.dtype, "output"), _ptr(ws), need,
                                  _stream(dev))
    if rc:
        _lib.check(rc, "sb_group4_linear")
    return y


def gated_mlp(x: torch.Tensor, gate: Group4Matrix, up: Group4Matrix, down: Group4Matrix, out_dtype=None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[..., H] = down(silu(gate x) * (up x)): gate and up [I, H], down [H, I]."""
    lib, dev = _lib.load(), gate.device
    if up.device != dev or down.device != dev:
        raise RuntimeError("gate, up and down must be on one device")
    x2, M, ldx = _rows(x, gate.K, dev)
    y = _output(out, (*x.shape[:-1], down.N), out_dtype or x.dtype, dev, activations=x2)
    xc = _code(x2.dtype, "activation")
    need = lib.sb_group4_gated_mlp_workspace_bytes(xc, M, gate.K, gate.N)
    ws = _workspace(need, dev)
    with _on(dev):
        rc = lib.sb_group4_gated_mlp(x2.data_ptr(), xc, ldx, M, gate.ref, up.ref, down.ref, y.data_ptr(),
                                     _code(y.dtype, "output"), ws.data_ptr(), need, _stream(dev))
    if rc:
        _lib.check(rc, "sb_group4_gated_mlp")
    return y


@functools.lru_cache(maxsize=None)
def max_tokens(top_k: int) -> int:
    """The most tokens of one few-token call (a larger batch is cut into such calls)."""
    return int(_lib.load().sb_moe_few_max_tokens(int(top_k)))


@functools.lru_cache(maxsize=1024)
def _moe_bytes(xc: int, B: int, H: int, I: int, E: int, k: int) -> int:
    return int(_lib.load().sb_moe_few_workspace_bytes(xc, B, H, I, E, k))


def few_moe(experts, x: torch.Tensor, ids: Optional[torch.Tensor], weights: Optional[torch.Tensor],
            gate_weight: Optional[torch.Tensor] = None, top_k: int = 0, norm_topk: bool = False, out_dtype=None,
            out: Optional[torch.Tensor] = None, routing: bool = True):
    """The few-token layer over ``experts`` (``TernaryExperts`` or ``Group4Experts``):
    (out, ids, weights).  With ``gate_weight`` [E, H] the routing is computed (and
    returned if ``routing``), else ids and weights [B, k] are given."""
    lib, dev, E, H = _lib.load(), experts.gate.device, experts.E, experts.H
    x2, B, ldx = _rows(x, H, dev)
    xc, gw, gc = _code(x2.dtype, "activation"), None, 0
    if gate_weight is None:
        _check_cuda(ids, "ids", dev)
        _check_cuda(weights, "weights", dev)
        _no_grad(weights, "the routing's weights")
        if ids.dim() != 2 or ids.shape[0] != B or ids.shape != weights.shape:
            raise RuntimeError(f"ids {tuple(ids.shape)} and weights {tuple(weights.shape)} must be [{B}, k]")
        k = ids.shape[1]
        if ids.dtype != torch.int32 or not ids.is_contiguous():
            if ids.dtype not in (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8):
                raise RuntimeError(f"ids must be whole numbers, got {ids.dtype}")
            ids = ids.to(torch.int64).clamp(-1, E).to(torch.int32).contiguous()  # (-1 and E are dropped and reported)
        if weights.dtype != torch.float32 or not weights.is_contiguous():
            weights = weights.detach().to(torch.float32).contiguous()
    else:
        _no_grad(gate_weight, "the gate's weights")
        _check_cuda(gate_weight, "gate_weight", dev)
        if gate_weight.shape != (E, H):
            raise RuntimeError(f"gate_weight of shape {tuple(gate_weight.shape)} must be [{E}, {H}]")
        gate_weight = gate_weight.contiguous()  # (copied only where it is not)
        k, gw, gc = top_k, gate_weight.data_ptr(), _code(gate_weight.dtype, "gate")
    most = max_tokens(k)
    if most < 1:
        raise RuntimeError(f"top_k {k} is not in 1..32")
    y = _output(out, x.shape, out_dtype or x.dtype, dev, activations=x2, ids=ids, weights=weights, gate_weights=gate_weight)
    yc, n = _code(y.dtype, "output"), min(B, most)
    need = _moe_bytes(xc, n, H, experts.I, E, k)
    if ids is not None:
        ip, wp, ws = ids.data_ptr(), weights.data_ptr(), _workspace(need, dev)
    elif routing or B > most:
        ids = torch.empty(B, k, dtype=torch.int32, device=dev)
        weights = torch.empty(B, k, dtype=torch.float32, device=dev)
        ip, wp, ws = ids.data_ptr(), weights.data_ptr(), _workspace(need, dev)
    else:  # nobody reads the routing: behind the workspace
        ws = _workspace(need + 8 * B * k, dev)
        ip = ws.data_ptr() + need
        wp = ip + 4 * B * k
    with _on(dev):
        stream, ref, xp, yp, wsp, norm = _stream(dev), experts.few_ref, x2.data_ptr(), y.data_ptr(), ws.data_ptr(), int(norm_topk)
        xb, yb = x2.element_size(), y.element_size()
        for b in range(0, B, most) if B else (0,):
            rc = lib.sb_moe_few(ref, xp + b * ldx * xb, xc, ldx, min(most, B - b), k, gw, gc, norm, ip + 4 * b * k,
                                wp + 4 * b * k, yp + b * H * yb, yc, wsp, need, stream)
            if rc:
                _lib.check(rc, "sb_moe_few")
    return y, ids, weights


def check_experts(E: int, H: int, I: int) -> None:
    """Experts that the few-token layer takes."""
    if E > MAX_EXPERTS or max(H, I) > MAX_WIDTH:
        raise RuntimeError(f"{E} experts of {H} x {I}: the few-token layer takes up to {MAX_EXPERTS} experts and {MAX_WIDTH} "
                           "channels each way")


class Group4Experts:
    """E SwiGLU experts in 4-bit groups on one device: ``gate`` and ``up`` count E
    matrices [I, H], ``down`` E matrices [H, I], all in groups of one size, with zero
    points in all three or in none.  E is at most ``MAX_EXPERTS``, H and I ``MAX_WIDTH``
    (``gated_mlp`` takes single experts of up to 16384)."""

    def __init__(self, gate: Group4Matrix, up: Group4Matrix, down: Group4Matrix):
        self.E, self.I, self.H = gate.count, gate.N, gate.K
        check_experts(self.E, self.H, self.I)
        if (up.count, up.N, up.K) != (self.E, self.I, self.H) or (down.count, down.N, down.K) != (self.E, self.H, self.I):
            raise RuntimeError(f"{gate.count} gate [{gate.N}, {gate.K}], {up.count} up [{up.N}, {up.K}] and {down.count} "
                               f"down [{down.N}, {down.K}] matrices are not experts of one shape")
        if len({m.group for m in (gate, up, down)}) > 1 or len({m.has_zeros for m in (gate, up, down)}) > 1:
            raise RuntimeError("gate, up and down must have one group size, and zero points in all three or in none")
        if len({m.device for m in (gate, up, down)}) > 1:
            raise RuntimeError("gate, up and down must be on one device")
        self.gate, self.up, self.down, self.device = gate, up, down, gate.device
        self.few_desc = _lib.Experts(_lib.SB_EXPERTS_GROUP4, self.E, self.H, self.I, gate.group, int(gate.has_zeros),
                                     gate.data.data_ptr(), up.data.data_ptr(), down.data.data_ptr(), None, None, None)
        self.few_ref = C.byref(self.few_desc)

    @classmethod
    def pack(cls, gate: dict, up: dict, down: dict, group: int = 128) -> "Group4Experts":
        """From codes [E, N, K], scales and (optional) zeros of each kind of matrix, as
        ``Group4Matrix.pack`` takes them."""
        shape = gate["codes"].shape
        if len(shape) > 1:
            check_experts(math.prod(shape[:-2]), shape[-1], shape[-2])
        return cls(*(Group4Matrix.pack(m["codes"], m["scales"], m.get("zeros"), group) for m in (gate, up, down)))

    @classmethod
    def quantize(cls, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, group: int = 128,
                 symmetric: bool = True) -> "Group4Experts":
        """From the experts' weights: gate and up [E, I, H], down [E, H, I]."""
        for t, what in ((gate, "gate"), (up, "up"), (down, "down")):
            if t.dim() != 3:
                raise RuntimeError(f"{what} must be [E, N, K], got {tuple(t.shape)}")
        check_experts(gate.shape[0], gate.shape[2], gate.shape[1])
        return cls(*(quantize(t, group, symmetric) for t in (gate, up, down)))

    def memory_bytes(self) -> int:
        return sum(m.memory_bytes() for m in (self.gate, self.up, self.down))

    def forward_few(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, out_dtype=torch.float32,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """out[t] = sum_j weights[t,j] * expert_{ids[t,j]}(x[t]) for a few tokens (more are
        cut into calls of ``max_tokens(k)``)."""
        return few_moe(self, x, ids, weights, out_dtype=out_dtype, out=out)[0]

    forward = forward_few
