"""Device-level operators: torch CUDA tensors in, torch CUDA tensors out, every one a
single call into the C ABI on torch's current stream.  torch is used for device
memory and streams only; no operator here has a PyTorch implementation."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


# torch.cuda.current_stream().cuda_stream without the Stream object in between (3.1 -> 0.2 us, of about 13 for an operator call
# whose kernel takes 3); the operators' tensors exist, so CUDA is initialised
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # (a torch built without CUDA can import this module)
_device = getattr(torch._C, "_cuda_getDevice", None)


def _stream():
    return _raw_stream(_device())


def _want(t: torch.Tensor, dtype, name: str):
    if not t.is_cuda:
        raise _lib.AwqBackendError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise _lib.AwqBackendError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise _lib.AwqBackendError(f"{name} must be contiguous")
    return t


def _aligned16(*tensors):
    return not any(t is not None and t.data_ptr() & 15 for t in tensors)


def _parts(size_fn: str, device, *dims):
    """Scratch that the kernel chosen for these sizes asks for, from torch's stream-ordered allocator; None where it needs none."""
    n = int(getattr(_lib.load(), size_fn)(*dims))
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


@dataclass
class AwqWeight:
    """One AWQ-quantised linear layer in HF AutoAWQ layout (layout A), resident on a GPU.

    qweight int32 [K, N/8], qzeros int32 [K/gs, N/8], scales bf16 [K/gs, N].
    """
    qweight: torch.Tensor
    qzeros: torch.Tensor
    scales: torch.Tensor
    group_size: int = 128

    def __post_init__(self):
        _want(self.qweight, torch.int32, "qweight")
        _want(self.qzeros, torch.int32, "qzeros")
        _want(self.scales, torch.bfloat16, "scales")
        K, nb = self.qweight.shape
        if self.qzeros.shape != (K // self.group_size, nb) or self.scales.shape != (K // self.group_size, nb * 8):
            raise _lib.AwqBackendError(
                f"qzeros {tuple(self.qzeros.shape)} / scales {tuple(self.scales.shape)} do not match "
                f"qweight {tuple(self.qweight.shape)} with group size {self.group_size}")

    @property
    def K(self):
        return self.qweight.shape[0]

    @property
    def N(self):
        return self.qweight.shape[1] * 8

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.qweight, self.qzeros, self.scales))

    @classmethod
    def from_numpy(cls, qweight, qzeros, scales, group_size=128, device="cuda"):
        """Host arrays (scales bf16 as ml_dtypes.bfloat16, or fp16/fp32 rounded to bf16 as
        awq_repacker.py:74-78 does) -> device-resident weight."""
        import numpy as np
        from ml_dtypes import bfloat16
        s = np.ascontiguousarray(np.asarray(scales).astype(bfloat16)).view(np.int16)
        return cls(torch.from_numpy(np.ascontiguousarray(qweight, dtype=np.int32)).to(device),
                   torch.from_numpy(np.ascontiguousarray(qzeros, dtype=np.int32)).to(device),
                   torch.from_numpy(s).to(device).view(torch.bfloat16), group_size)


class Workspace:
    """Caller-owned scratch for the decode kernels (strip counters + split-K partials).
    One per stream: calls that share a workspace must not overlap on the GPU."""

    def __init__(self, K: int, N: int, device="cuda", batch: int = 64):
        self.nbytes = int(_lib.load().awq_b200_workspace_bytes(int(batch), int(K), int(N)))
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        with torch.cuda.device(self.buf.device):
            _lib.call("awq_b200_workspace_init", self.buf.data_ptr(), self.nbytes, _stream())

    def fits(self, K, N, batch=64):
        return int(_lib.load().awq_b200_workspace_bytes(int(batch), int(K), int(N))) <= self.nbytes

    def check(self):
        """Synchronise and raise if a device-side wait timed out."""
        with torch.cuda.device(self.buf.device):
            _lib.call("awq_b200_workspace_check", self.buf.data_ptr(), _stream())
            _lib.call("awq_b200_gemm_check", _stream())  # gemv of more than 8 rows: the batched-decode GEMM's waits


ACT_BF16, ACT_F16, OUT_F32 = 0, 1, 2


def _act_dtype(f16: bool):
    return torch.float16 if f16 else torch.bfloat16


def set_decode_kernel(mode: str):
    """"auto", "generic", "streamk" (fp16 activation path) or "streamk_bf16" (bf16 activations as they are)."""
    _lib.call("awq_b200_set_decode_kernel", {"auto": 0, "generic": 1, "streamk": 2, "streamk_bf16": 3}[mode])


def set_deterministic(on: bool):
    """Kept for callers of earlier versions; a no-op: split-K partials are summed as integers, so every result is
    bit-reproducible already."""
    _lib.call("awq_b200_set_deterministic", 1 if on else 0)


def set_gemm_kernel(mode: str):
    """"auto", "generic", or the tensor-core kernel where it covers the shape, an error elsewhere ("tc"; "tm" is the same)."""
    _lib.call("awq_b200_set_gemm_kernel", {"auto": 0, "generic": 1, "tc": 2, "tm": 3}[mode])


def dequant(w: AwqWeight, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """bf16 [K, N] = (q - z) * s, bit-exact with awq_repacker.dequant_to_bf16."""
    if out is None:
        out = torch.empty((w.K, w.N), dtype=torch.bfloat16, device=w.qweight.device)
    _want(out, torch.bfloat16, "out")
    _lib.call("awq_b200_dequant_bf16", _ptr(w.qweight), _ptr(w.qzeros), _ptr(w.scales), _ptr(out), w.K, w.N,
              w.group_size, _stream())
    return out


def dequant_1d(packed_q, scales, zeros, n, group_size, out=None):
    if out is None:
        out = torch.empty(n, dtype=torch.bfloat16, device=packed_q.device)
    _lib.call("awq_b200_dequant_1d_bf16", _ptr(_want(packed_q, torch.uint8, "packed_q")),
              _ptr(_want(scales, torch.bfloat16, "scales")), _ptr(_want(zeros, torch.uint8, "zeros")), _ptr(out),
              int(n), int(group_size), _stream())
    return out


def _x2d(x, K, f16=False):
    _want(x, _act_dtype(f16), "x")
    if x.dim() == 1:
        x = x.view(1, -1)
    if x.dim() != 2 or x.shape[1] != K:
        raise _lib.AwqBackendError(f"x must be [B, {K}], got {tuple(x.shape)}")
    return x


# From how many weights on bf16 gemv calls of 9 to 16 and of 17 to 64 rows take the fp8-operand GEMM: it is three launches where the
# multi-row GEMV kernel is two, and 3 us more for the host.  Measured per call, multi-row GEMV / GEMM: 32 rows, 45 M weights
# 25.2 / 18.7 us; 64 rows, 235 M 143 / 84; 24 rows, 15 M 18.2 / 18.9; 16 rows, 45 M 16.0 / 18.6, and per 70B layer in a graph 108 / 86.
GEMV_ROWS_MIN_WEIGHTS = {16: 100e6, 64: 32e6}


def gemv(x, w: AwqWeight, ws: Workspace, residual=None, out=None, f32_out=False, x_f16=False):
    """y [B, N] = x [B, K] @ W (+ residual); bf16 with one rounding, or the f32 partial.
    x is bf16, or fp16 (the library's internal activation format) with x_f16.  bf16 rows are multiplied as they are or as
    fp16; more than 8 rows on large weights (GEMV_ROWS_MIN_WEIGHTS) as two fp8 pieces, exact for an element from 2^-13 of the
    largest magnitude in its row's quantisation group on, smaller ones to 2^-21 of that magnitude."""
    x = _x2d(x, w.K, x_f16)
    B = x.shape[0]
    if out is None:
        out = torch.empty((B, w.N), dtype=torch.float32 if f32_out else torch.bfloat16, device=x.device)
    if f32_out and residual is not None:
        raise _lib.AwqBackendError("f32 partial output takes no residual")
    if residual is not None:
        _want(residual, torch.bfloat16, "residual")
    _want(out, torch.float32 if f32_out else torch.bfloat16, "out")
    if B > 8 and not x_f16 and w.K * w.N >= GEMV_ROWS_MIN_WEIGHTS[16 if B <= 16 else 64] and _aligned16(x, w.qweight, w.qzeros, w.scales, residual, out):
        scratch = _parts("awq_b200_gemv_rows_workspace_bytes", out.device, B, w.K, w.N, w.group_size)
        if scratch is not None:
            _lib.call("awq_b200_gemv_rows_bf16", _ptr(x), _ptr(w.qweight), _ptr(w.qzeros), _ptr(w.scales), _ptr(residual), _ptr(out),
                      1 if f32_out else 0, B, w.K, w.N, w.group_size, _ptr(scratch), scratch.numel(), _stream())
            return out
    _lib.call("awq_b200_gemv_act", _ptr(x), ACT_F16 if x_f16 else ACT_BF16, _ptr(w.qweight), _ptr(w.qzeros),
              _ptr(w.scales), _ptr(residual), _ptr(out), 1 if f32_out else 0, B, w.K, w.N, w.group_size, _ptr(ws.buf),
              ws.nbytes, _stream())
    return out


def gateup_swiglu(x, w_gateup: AwqWeight, ws: Workspace, out=None, x_f16=False, out_f16=False):
    """out [B, I] = silu(gate) * up for a gate/up-interleaved [K, 2I] weight."""
    x = _x2d(x, w_gateup.K, x_f16)
    B, I = x.shape[0], w_gateup.N // 2
    if out is None:
        out = torch.empty((B, I), dtype=_act_dtype(out_f16), device=x.device)
    _lib.call("awq_b200_gateup_swiglu_act", _ptr(x), ACT_F16 if x_f16 else ACT_BF16, _ptr(w_gateup.qweight),
              _ptr(w_gateup.qzeros), _ptr(w_gateup.scales), _ptr(_want(out, _act_dtype(out_f16), "out")),
              ACT_F16 if out_f16 else ACT_BF16, B, w_gateup.K, I, w_gateup.group_size, _ptr(ws.buf), ws.nbytes, _stream())
    return out


def interleave_gate_up(gate: AwqWeight, up: AwqWeight) -> AwqWeight:
    """Two [K, I] weights -> one [K, 2I] weight with column 2i = gate_i, 2i+1 = up_i."""
    if (gate.K, gate.N, gate.group_size) != (up.K, up.N, up.group_size):
        raise _lib.AwqBackendError("gate and up must have the same shape and group size")
    K, I, G = gate.K, gate.N, gate.K // gate.group_size
    dev = gate.qweight.device
    qw = torch.empty((K, 2 * I // 8), dtype=torch.int32, device=dev)
    qz = torch.empty((G, 2 * I // 8), dtype=torch.int32, device=dev)
    sc = torch.empty((G, 2 * I), dtype=torch.bfloat16, device=dev)
    _lib.call("awq_b200_interleave_gate_up", _ptr(gate.qweight), _ptr(gate.qzeros), _ptr(gate.scales),
              _ptr(up.qweight), _ptr(up.qzeros), _ptr(up.scales), _ptr(qw), _ptr(qz), _ptr(sc), K, I,
              gate.group_size, _stream())
    return AwqWeight(qw, qz, sc, gate.group_size)


def rmsnorm(x, gamma, eps=1e-5, out=None, out_f16=False):
    _want(x, torch.bfloat16, "x")
    x2 = x.view(1, -1) if x.dim() == 1 else x
    if out is None:
        out = torch.empty(x2.shape, dtype=_act_dtype(out_f16), device=x.device)
    _lib.call("awq_b200_rmsnorm_act", _ptr(x2), _ptr(_want(gamma, torch.bfloat16, "gamma")), float(eps),
              _ptr(_want(out, _act_dtype(out_f16), "out")), ACT_F16 if out_f16 else ACT_BF16, x2.shape[0], x2.shape[1],
              _stream())
    return out


def add_rmsnorm(h, partial_sum, gamma=None, eps=1e-5, h_out=None, normed=None, normed_f16=False):
    """h_out = bf16(h + partial_sum); normed = rmsnorm(h_out, gamma) when gamma is given."""
    _want(h, torch.bfloat16, "h")
    _want(partial_sum, torch.float32, "partial_sum")
    if h_out is None:
        h_out = torch.empty_like(h)
    if gamma is not None and normed is None:
        normed = torch.empty(h.shape, dtype=_act_dtype(normed_f16), device=h.device)
    _lib.call("awq_b200_add_rmsnorm_act", _ptr(h), _ptr(partial_sum), _ptr(gamma), float(eps), _ptr(h_out),
              _ptr(normed), ACT_F16 if normed_f16 else ACT_BF16, h.shape[0], h.shape[1], _stream())
    return h_out, normed


def ffn_decode(x, w_gateup: AwqWeight, w_down: AwqWeight, ws: Workspace, gamma=None, eps=1e-5, residual=None,
               normed=None, inter=None, out=None):
    """out [B, H] = down(swiglu(gateup . norm(x))) (+ residual): one C-ABI call, three kernels.
    `normed` and `inter` are 16-bit scratch (the library keeps its intermediates there as fp16)."""
    x = _x2d(x, w_gateup.K)
    B, H, I = x.shape[0], w_gateup.K, w_gateup.N // 2
    if w_down.K != I or w_down.N != H:
        raise _lib.AwqBackendError(f"down weight must be [{I}, {H}], got [{w_down.K}, {w_down.N}]")
    dev = x.device
    if gamma is not None and normed is None:
        normed = torch.empty((B, H), dtype=torch.float16, device=dev)
    if inter is None:
        inter = torch.empty((B, I), dtype=torch.float16, device=dev)
    if out is None:
        out = torch.empty((B, H), dtype=torch.bfloat16, device=dev)
    _lib.call("awq_b200_ffn_decode_bf16", _ptr(x), _ptr(gamma), float(eps), _ptr(w_gateup.qweight),
              _ptr(w_gateup.qzeros), _ptr(w_gateup.scales), _ptr(w_down.qweight), _ptr(w_down.qzeros),
              _ptr(w_down.scales), _ptr(residual), _ptr(normed), _ptr(inter), _ptr(out), B, H, I, w_gateup.group_size,
              _ptr(ws.buf), ws.nbytes, _stream())
    return out


def gemv_f32_push(x, w: AwqWeight, ws: Workspace, peers, slot: int, x_f16=False):
    """This rank's f32 partial x @ w written to its send slot, every rank signalled
    (`peers`: mlir_air_b200.peer.PeerBuffers); B <= 8."""
    x = _x2d(x, w.K, x_f16)
    _lib.call("awq_b200_gemv_f32_push", _ptr(x), ACT_F16 if x_f16 else ACT_BF16, _ptr(w.qweight), _ptr(w.qzeros),
              _ptr(w.scales), peers.local_send(slot), x.shape[0], w.K, w.N, w.group_size, peers.flag_array(slot),
              peers.world, peers.rank, _ptr(ws.buf), ws.nbytes, _stream())


def tp_reduce_add_rmsnorm(h, peers, slot: int, ws: Workspace, gamma=None, eps=1e-5, h_out=None, normed=None,
                          normed_f16=False):
    """Wait for every rank's partial in `slot`, h_out = bf16(h + sum of the partials in rank order),
    and with gamma the RMSNorm of h_out."""
    _want(h, torch.bfloat16, "h")
    if h_out is None:
        h_out = torch.empty_like(h)
    if gamma is not None and normed is None:
        normed = torch.empty(h.shape, dtype=_act_dtype(normed_f16), device=h.device)
    _lib.call("awq_b200_tp_reduce_add_rmsnorm_act", _ptr(h), peers.send_array(slot), peers.local_flags(slot),
              peers.world, _ptr(gamma), float(eps), _ptr(h_out), _ptr(normed), ACT_F16 if normed_f16 else ACT_BF16,
              h.shape[0], h.shape[1], _ptr(ws.buf), _stream())
    return h_out, normed


class FFNStackPlan:
    """Tensor maps of a decode FFN layer stack in device memory, for ffn_stack_decode.
    `gateups`, `downs`: one AwqWeight per layer (gate/up interleaved [H, 2I], down [I, H]);
    `gammas`: one bf16 [H] tensor per layer.  Keeps references to the weights it describes."""

    def __init__(self, gateups: Sequence[AwqWeight], downs: Sequence[AwqWeight], gammas: Sequence[torch.Tensor]):
        import ctypes
        n = len(gateups)
        if n == 0 or len(downs) != n or len(gammas) != n:
            raise _lib.AwqBackendError("FFNStackPlan: one gate/up weight, one down weight and one gamma per layer")
        self.n_layers = n
        self.H, self.I, self.group_size = gateups[0].K, gateups[0].N // 2, gateups[0].group_size
        for gu, d, g in zip(gateups, downs, gammas):
            if (gu.K, gu.N, d.K, d.N, gu.group_size, d.group_size) != (self.H, 2 * self.I, self.I, self.H, self.group_size,
                                                                         self.group_size):
                raise _lib.AwqBackendError("FFNStackPlan: all layers must have the same shape and group size")
            _want(g, torch.bfloat16, "gamma")
            if g.numel() != self.H:
                raise _lib.AwqBackendError(f"FFNStackPlan: gamma must have {self.H} elements")
        self._keep = (list(gateups), list(downs), list(gammas))
        dev = gateups[0].qweight.device
        lib = _lib.load()
        self.nbytes = int(lib.awq_b200_ffn_stack_plan_bytes(n))
        self.buf = torch.empty(self.nbytes + 128, dtype=torch.uint8, device=dev)
        self.ptr = (self.buf.data_ptr() + 127) // 128 * 128
        arr = ctypes.c_void_p * n

        def ptrs(ts):
            return arr(*[t.data_ptr() for t in ts])

        with torch.cuda.device(dev):
            _lib.call("awq_b200_ffn_stack_plan", self.ptr, self.nbytes, n, ptrs([w.qweight for w in gateups]),
                      ptrs([w.qzeros for w in gateups]), ptrs([w.scales for w in gateups]), ptrs([w.qweight for w in downs]),
                      ptrs([w.qzeros for w in downs]), ptrs([w.scales for w in downs]), ptrs(list(gammas)), self.H, self.I,
                      self.group_size)

    def workspace_bytes(self) -> int:
        return int(_lib.load().awq_b200_ffn_stack_workspace_bytes(self.n_layers))


def set_ffn_stack_tuning(lookahead_units: int = -1, split_per_1024: int = -1):
    """Tuning of the one-launch stack kernel (negative = keep): units per half-CTA prefetched into
    L2 ahead of the ring; and 0 = a down unit waits for the whole gate/up phase, other = only for the
    sub-strips that produce its inputs (the default)."""
    _lib.call("awq_b200_set_ffn_stack_tuning", int(lookahead_units), int(split_per_1024))


def ffn_stack_decode(plan: FFNStackPlan, x, ws: Workspace, eps=1e-5, inter=None, out=None):
    """out [B, H] = the whole layer stack applied to x [B <= 8, H], ONE kernel launch."""
    x = _x2d(x, plan.H)
    B = x.shape[0]
    if inter is None:
        inter = torch.empty((B, plan.I), dtype=torch.float16, device=x.device)
    if out is None:
        out = torch.empty((B, plan.H), dtype=torch.bfloat16, device=x.device)
    _want(out, torch.bfloat16, "out")
    if inter.numel() < B * plan.I or inter.element_size() != 2:
        raise _lib.AwqBackendError("ffn_stack_decode: inter must hold B * I 16-bit elements")
    _lib.call("awq_b200_ffn_stack_decode_bf16", plan.ptr, plan.n_layers, _ptr(x), _ptr(out), _ptr(inter), float(eps), B,
              plan.H, plan.I, plan.group_size, _ptr(ws.buf), ws.nbytes, _stream())
    return out


def ffn_stack_tp_slot_bytes(H: int, n_ranks: int) -> int:
    return int(_lib.load().awq_b200_ffn_stack_tp_slot_bytes(int(H), int(n_ranks)))


def ffn_stack_decode_tp(plan: FFNStackPlan, x, ws: Workspace, peers, eps=1e-5, inter=None, out=None):
    """The one-launch stack on this rank's shards, with the partials exchanged through `peers`
    (mlir_air_b200.peer.PeerBuffers with two slots of ffn_stack_tp_slot_bytes(H, world) bytes, used by
    nothing else and always with the same number of layers)."""
    x = _x2d(x, plan.H)
    B = x.shape[0]
    if inter is None:
        inter = torch.empty((B, plan.I), dtype=torch.float16, device=x.device)
    if out is None:
        out = torch.empty((B, plan.H), dtype=torch.bfloat16, device=x.device)
    _want(out, torch.bfloat16, "out")
    if inter.numel() < B * plan.I or inter.element_size() != 2:
        raise _lib.AwqBackendError("ffn_stack_decode_tp: inter must hold B * I 16-bit elements")
    _lib.call("awq_b200_ffn_stack_decode_tp_bf16", plan.ptr, plan.n_layers, _ptr(x), _ptr(out), _ptr(inter), float(eps), B,
              plan.H, plan.I, plan.group_size, peers.base_array(), peers.stride, peers.recv_bytes, peers.world, peers.rank,
              _ptr(ws.buf), ws.nbytes, _stream())
    return out


def gemm(A, w: AwqWeight, out=None, residual=None, swiglu=False):
    """C [M, N] = A [M, K] @ W, f32 accumulate, bf16 out (prefill).  With `residual` [M, N] the sum is
    bf16(acc + residual); with `swiglu` W is gate/up-interleaved and C is [M, N/2]."""
    _want(A, torch.bfloat16, "A")
    if A.dim() != 2 or A.shape[1] != w.K:
        raise _lib.AwqBackendError(f"A must be [M, {w.K}], got {tuple(A.shape)}")
    if residual is not None or swiglu:
        n_out = w.N // 2 if swiglu else w.N
        if out is None:
            out = torch.empty((A.shape[0], n_out), dtype=torch.bfloat16, device=A.device)
        _want(out, torch.bfloat16, "out")
        if residual is not None:
            _want(residual, torch.bfloat16, "residual")
        ws = _parts("awq_b200_gemm_workspace_bytes", out.device, A.shape[0], w.K, w.N, w.group_size)
        if ws is not None:
            _lib.call("awq_b200_gemm_ws_bf16", _ptr(A), _ptr(w.qweight), _ptr(w.qzeros), _ptr(w.scales), _ptr(residual), _ptr(out),
                      1 if swiglu else 0, A.shape[0], w.K, w.N, w.group_size, _ptr(ws), ws.numel(), _stream())
            return out
        _lib.call("awq_b200_gemm_fused_bf16", _ptr(A), _ptr(w.qweight), _ptr(w.qzeros), _ptr(w.scales), _ptr(residual),
                  _ptr(out), 1 if swiglu else 0, A.shape[0], w.K, w.N, w.group_size, _stream())
        return out
    if out is None:
        out = torch.empty((A.shape[0], w.N), dtype=torch.bfloat16, device=A.device)
    ws = _parts("awq_b200_gemm_workspace_bytes", out.device, A.shape[0], w.K, w.N, w.group_size)
    if ws is not None:
        _lib.call("awq_b200_gemm_ws_bf16", _ptr(A), _ptr(w.qweight), _ptr(w.qzeros), _ptr(w.scales), None, _ptr(out), 0, A.shape[0],
                  w.K, w.N, w.group_size, _ptr(ws), ws.numel(), _stream())
        return out
    _lib.call("awq_b200_gemm_bf16", _ptr(A), _ptr(w.qweight), _ptr(w.qzeros), _ptr(w.scales), _ptr(out), A.shape[0],
              w.K, w.N, w.group_size, _stream())
    return out


class GemmDecodeWorkspace:
    """Caller-owned scratch of `gemm_decode` (the f32 sums of each SM's share of a tile) for up to `batch` rows and `N`
    columns.  One per stream: calls that share it must not overlap on the GPU."""

    def __init__(self, N: int, device="cuda", batch: int = 64, K: int = 0):
        """`K` > 0 also makes room for the split token rows of `gemm_decode(..., f8=True)` and of `ffn_layer_decode`."""
        self.batch, self.N, self.K = int(batch), int(N), int(K)
        lib = _lib.load()
        self.nbytes = int(lib.awq_b200_gemm_decode_workspace_bytes(self.batch, self.N))
        if self.K > 0:
            self.nbytes = max(self.nbytes, int(lib.awq_b200_gemm_decode_f8_workspace_bytes(min(self.batch, 32), self.K, self.N)),
                              int(lib.awq_b200_ffn_layer_decode_workspace_bytes(min(self.batch, 64), self.K, (self.N + 1) // 2)))
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)

    def fits(self, M, N):
        return int(_lib.load().awq_b200_gemm_decode_workspace_bytes(int(M), int(N))) <= self.nbytes

    def fits_layer(self, M, H, I):
        return 0 < int(_lib.load().awq_b200_ffn_layer_decode_workspace_bytes(int(M), int(H), int(I))) <= self.nbytes

    def fits_f8(self, M, K, N):
        return int(M) <= 32 and 0 < int(_lib.load().awq_b200_gemm_decode_f8_workspace_bytes(int(M), int(K), int(N))) <= self.nbytes


def gemm_decode(A, w: AwqWeight, ws: GemmDecodeWorkspace, out=None, residual=None, swiglu=False, f32_out=False, out_f16=False,
                f8=False):
    """C [M, N] = A [M, K] @ W for a decode batch of M <= 64 rows (weights streamed once, all SMs busy whatever the
    shape); `residual` / `swiglu` as in `gemm`; `f32_out`: the f32 sums themselves (a tensor-parallel partial).
    A may be bf16 or fp16 (the weights are then dequantised to fp16 too: 11 significant bits instead of 8);
    `out_f16` stores a plain or SwiGLU result as fp16 for a following fp16 product.  `f8` (up to 32 rows): the kernel that
    feeds the tensor core the packed nibbles and split token rows as fp8 and applies zero point and scale in f32."""
    if A.dtype not in (torch.bfloat16, torch.float16):
        raise _lib.AwqBackendError(f"A must be bf16 or fp16, got {A.dtype}")
    _want(A, A.dtype, "A")
    if A.dim() != 2 or A.shape[1] != w.K:
        raise _lib.AwqBackendError(f"A must be [M, {w.K}], got {tuple(A.shape)}")
    if f32_out and (residual is not None or swiglu or out_f16):
        raise _lib.AwqBackendError("gemm_decode: f32_out takes neither residual, swiglu nor out_f16")
    if out_f16 and residual is not None:
        raise _lib.AwqBackendError("gemm_decode: the residual add goes with a bf16 output")
    dt = torch.float32 if f32_out else _act_dtype(out_f16)
    if out is None:
        out = torch.empty((A.shape[0], w.N // 2 if swiglu else w.N), dtype=dt, device=A.device)
    _want(out, dt, "out")
    if residual is not None:
        _want(residual, torch.bfloat16, "residual")
    _lib.call("awq_b200_gemm_decode_f8" if f8 else "awq_b200_gemm_decode_act", _ptr(A), ACT_F16 if A.dtype == torch.float16 else ACT_BF16, _ptr(w.qweight),
              _ptr(w.qzeros), _ptr(w.scales), _ptr(residual), _ptr(out), OUT_F32 if f32_out else (ACT_F16 if out_f16 else ACT_BF16),
              1 if swiglu else 0, A.shape[0], w.K, w.N, w.group_size, _ptr(ws.buf), ws.nbytes, _stream())
    return out


def ffn_layer_decode(x, w_gateup: AwqWeight, w_down: AwqWeight, ws: GemmDecodeWorkspace, gamma, eps=1e-5, out=None):
    """out [B, H] = bf16(x + down(swiglu(gateup . rmsnorm(x, gamma)))) for a decode batch of up to 64 rows: one call, five
    launches (norm, product, SwiGLU, product, residual add).  Between the kernels the bf16 values of up to 32 rows are two fp8
    pieces each (bounds as in `gemv`) and no weight is rounded; more rows are fp16, and so are the weights."""
    x = _x2d(x, w_gateup.K)
    B, H, I = x.shape[0], w_gateup.K, w_gateup.N // 2
    if w_down.K != I or w_down.N != H:
        raise _lib.AwqBackendError(f"down weight must be [{I}, {H}], got [{w_down.K}, {w_down.N}]")
    if w_down.group_size != w_gateup.group_size:
        raise _lib.AwqBackendError(f"both weights must have one group size, got {w_gateup.group_size} and {w_down.group_size}")
    if gamma.numel() != H:
        raise _lib.AwqBackendError(f"gamma must have {H} elements, got {gamma.numel()}")
    if out is None:
        out = torch.empty((B, H), dtype=torch.bfloat16, device=x.device)
    if tuple(out.shape) != (B, H) and not (B == 1 and tuple(out.shape) == (H,)):
        raise _lib.AwqBackendError(f"out must be [{B}, {H}], got {tuple(out.shape)}")
    _lib.call("awq_b200_ffn_layer_decode_bf16", _ptr(x), _ptr(_want(gamma, torch.bfloat16, "gamma")), float(eps), _ptr(w_gateup.qweight),
              _ptr(w_gateup.qzeros), _ptr(w_gateup.scales), _ptr(w_down.qweight), _ptr(w_down.qzeros), _ptr(w_down.scales),
              _ptr(_want(out, torch.bfloat16, "out")), B, H, I, w_gateup.group_size, _ptr(ws.buf), ws.nbytes, _stream())
    return out


def rope_halfsplit(x, lut, n_heads: int, head_dim: int, out=None):
    """Half-split RoPE of x [B, >= n_heads * head_dim] (a column slice of a wider projection output
    is fine: the row stride is passed on) with one LUT row [cos | sin] per token; in place by default."""
    _want(lut, torch.bfloat16, "lut")
    if out is None:
        out = x
    for name, t in (("x", x), ("out", out)):
        if not t.is_cuda or t.dtype != torch.bfloat16 or t.dim() != 2 or t.stride(1) != 1 or \
                t.shape[1] < n_heads * head_dim:
            raise _lib.AwqBackendError(f"rope: {name} must be a CUDA bf16 [B, >= n_heads * head_dim] tensor with unit "
                                       "column stride")
    if out.shape[0] != x.shape[0] or lut.shape != (x.shape[0], head_dim):
        raise _lib.AwqBackendError(f"rope: out must have {x.shape[0]} rows and lut must be [{x.shape[0]}, {head_dim}]")
    # the stride of a one-row tensor is arbitrary (0 after numpy's None indexing): it is never used
    xs = x.stride(0) if x.shape[0] > 1 else n_heads * head_dim
    os_ = out.stride(0) if out.shape[0] > 1 else n_heads * head_dim
    _lib.call("awq_b200_rope_halfsplit_bf16", x.data_ptr(), xs, _ptr(lut), out.data_ptr(), os_, x.shape[0], n_heads,
              head_dim, _stream())
    return out


# ---- many requests: paged cache, drafted tokens, adapters -----------------------------------------------------------------
def _on(t: torch.Tensor, name: str, dtype, device: int, dim: int = 1):
    """`t` as an argument on `device`: its type, its dimensions, its values side by side."""
    if t.dtype is dtype and t.get_device() == device and t.dim() == dim and t.is_contiguous():
        return t.data_ptr()
    if t.dtype != dtype or t.dim() != dim or t.get_device() != device:
        raise _lib.AwqBackendError(f"{name} must be a {dim}-dimensional {dtype} tensor on cuda:{device}, got {t.dim()} dimensions of {t.dtype} "
                                   f"on {t.device}")
    raise _lib.AwqBackendError(f"{name} must be contiguous")


def _sizes(**want):
    """Raises for the first (tensor, elements) that does not fit."""
    for name, (t, n) in want.items():
        if t.numel() != n:
            raise _lib.AwqBackendError(f"{name} must have {n} elements, got {t.numel()}")


def _call_on(device: int, name: str, *args):
    """The call on `device`'s current stream, whichever device is the current one."""
    if device == _device():
        return _lib.call(name, *args, _raw_stream(device))
    with torch.cuda.device(device):
        return _lib.call(name, *args, _raw_stream(device))


class RequestWorkspace:
    """Scratch and error word of the operators on many requests' rows (`page_plan`, `rope_append`, `tree_attention`, `page_keep`,
    `lora`); one size serves them all.  One per stream: calls that share it must not overlap on the GPU, nor may graphs
    captured with it."""

    def __init__(self, device="cuda"):
        self.nbytes = int(_lib.load().awq_b200_request_workspace_bytes())
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)
        if not self.buf.is_cuda:
            raise _lib.AwqBackendError("RequestWorkspace needs a CUDA device")
        self.ptr, self.device = self.buf.data_ptr(), self.buf.get_device()
        _call_on(self.device, "awq_b200_workspace_init", self.ptr, self.nbytes)

    def check(self):
        """Synchronise and raise if a call since the last check met a length, page, slot, path or adapter outside its buffers."""
        _call_on(self.device, "awq_b200_request_check", self.ptr)


class KVCache:
    """K and V of one layer in pages: [n_pages, page_size, n_kv_heads, head_dim] each, bf16 or fp16.  Views with other strides
    (heads in front of slots, K and V in one tensor) are fine as long as a head's values lie side by side and all strides are
    multiples of 8 elements.  Checked once, here; keeps the tensors alive."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        for name, t in (("k", k), ("v", v)):
            if not t.is_cuda or t.dtype not in (torch.bfloat16, torch.float16) or t.dim() != 4:
                raise _lib.AwqBackendError(f"KVCache: {name} must be a bf16 or fp16 CUDA tensor [n_pages, page_size, n_kv_heads, head_dim]")
            if t.numel() == 0 or t.stride(3) != 1 or any(t.stride(i) % 8 or t.stride(i) <= 0 for i in range(3) if t.shape[i] > 1):
                raise _lib.AwqBackendError(f"KVCache: {name} needs elements, a unit stride over head_dim and positive multiples of 8 elsewhere")
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise _lib.AwqBackendError("KVCache: k and v must have the same shape, type and device")
        self.k, self.v, self.dtype, self.device = k, v, k.dtype, k.get_device()
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k.shape
        if self.n_pages * self.page_size > 0x7fffffff:
            raise _lib.AwqBackendError("KVCache: more than 2^31 - 1 slots")
        if self.head_dim % 16 or self.head_dim > 256:
            raise _lib.AwqBackendError(f"KVCache: head_dim must be a multiple of 16, at most 256, got {self.head_dim}")
        if not _aligned16(k, v):
            raise _lib.AwqBackendError("KVCache: k and v must be 16-byte aligned")
        strides = [t.stride(i) if t.shape[i] > 1 else 0 for t in (k, v) for i in range(3)]
        self._struct = _lib.KvCacheStruct(k.data_ptr(), v.data_ptr(), *strides, self.n_pages, self.page_size, self.n_kv_heads, self.head_dim,
                                          ACT_F16 if k.dtype == torch.float16 else ACT_BF16)
        self.ptr = _lib.address_of(self._struct)

    def rows(self, t: torch.Tensor, name: str, n_heads=None, rows=None):
        """Checks [T, heads, head_dim] rows that go with the cache (column slices of a wider projection are fine)."""
        if t.dim() != 3 or t.dtype is not self.dtype or t.get_device() != self.device:
            raise _lib.AwqBackendError(f"{name} must be [T, heads, {self.head_dim}] of {self.dtype} on cuda:{self.device}, got {tuple(t.shape)} of {t.dtype} on {t.device}")
        T, heads, dim = t.shape
        row, head, unit = t.stride()
        if dim != self.head_dim or unit != 1 or (n_heads is not None and heads != n_heads) or (rows is not None and T != rows):
            raise _lib.AwqBackendError(f"{name} must be [{'T' if rows is None else rows}, {'heads' if n_heads is None else n_heads}, {self.head_dim}] with unit "
                                       f"stride over head_dim, got {tuple(t.shape)}")
        # the stride of a dimension of one is arbitrary and never used
        return t.data_ptr(), row if T > 1 else 0, head if heads > 1 else 0


@dataclass
class StepPlan:
    """The rows of one step, from `page_plan`: q_start int32 [R + 1], slots and positions int32 [T], mask int64 [T] or None."""
    q_start: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    mask: Optional[torch.Tensor] = None


def _table(table: torch.Tensor, R: int, device: int):
    if table.dtype is torch.int32 and table.dim() == 2 and table.get_device() == device:
        (rows, width), (stride, unit) = table.shape, table.stride()
        if rows == R and (unit == 1 or width <= 1):
            return table.data_ptr(), stride if R > 1 else width, width
    raise _lib.AwqBackendError(f"table must be int32 [{R}, width] on cuda:{device} with unit column stride, got {tuple(table.shape)} of {table.dtype}")


def page_plan(lens, new, table, free_pages, free_count, page_size: int, T: int, ws: RequestWorkspace, parents=None, free_count_out=None,
              out: Optional[StepPlan] = None) -> StepPlan:
    """Plan a step of `T` rows: every request r has lens[r] tokens in the cache and brings new[r] more.  Pages for them are popped
    from `free_pages` (a stack of free_count[0] page numbers) into `table` int32 [R, width], request by request; the plan says
    each row's request, slot and position and, with `parents` (int32, per row the index in its tree of the token it continues,
    -1: the last cached one; at most 64 per request), the mask of its ancestors.  free_count is updated in place unless
    free_count_out is given; lens stays: `page_keep` moves it on.  A step that does not fit changes nothing, has no rows, and
    ws.check() says so; rows behind the last request get slot -1."""
    dev, R, i32 = ws.device, lens.numel(), torch.int32
    count_out = free_count if free_count_out is None else free_count_out
    lens_p, new_p, free_p, count_p, count_out_p = (_on(lens, "lens", i32, dev), _on(new, "new", i32, dev), _on(free_pages, "free_pages", i32, dev),
                                                   _on(free_count, "free_count", i32, dev), _on(count_out, "free_count_out", i32, dev))
    table_p, stride, width = _table(table, R, dev)
    if new.numel() != R or free_count.numel() != 1 or count_out.numel() != 1:
        _sizes(new=(new, R), free_count=(free_count, 1), free_count_out=(count_out, 1))
    if out is None:  # one allocation, three views of it
        rows = torch.empty(R + 1 + 2 * T, dtype=i32, device=lens.device)
        out = StepPlan(*rows.split((R + 1, T, T)), None if parents is None else torch.empty(T, dtype=torch.int64, device=lens.device))
    parents_p = mask_p = None
    if parents is not None:
        parents_p = _on(parents, "parents", i32, dev)
        if out.mask is None:
            raise _lib.AwqBackendError("page_plan: parents need a mask in `out`")
        mask_p = _on(out.mask, "out.mask", torch.int64, dev)
        if parents.numel() != T or out.mask.numel() != T:
            _sizes(parents=(parents, T), mask=(out.mask, T))
    elif out.mask is not None:
        raise _lib.AwqBackendError("page_plan: a mask in `out` needs parents")
    start_p, slots_p, pos_p = _on(out.q_start, "out.q_start", i32, dev), _on(out.slots, "out.slots", i32, dev), _on(out.positions, "out.positions", i32, dev)
    if out.q_start.numel() != R + 1 or out.slots.numel() != T or out.positions.numel() != T:
        _sizes(q_start=(out.q_start, R + 1), slots=(out.slots, T), positions=(out.positions, T))
    _call_on(dev, "awq_b200_page_plan", lens_p, new_p, table_p, stride, width, free_p, free_pages.numel(), count_p, count_out_p, parents_p,
             int(page_size), start_p, slots_p, pos_p, mask_p, R, T, ws.ptr, ws.nbytes)
    return out


def rope_append(q, k, v, lut, positions, slots, cache: KVCache, ws: RequestWorkspace, q_out=None):
    """Half-split RoPE of q [T, n_heads, head_dim] (in place, or into q_out) and k [T, n_kv_heads, head_dim] by the rows
    positions[t] of lut bf16 [n_positions, head_dim] ([cos | sin], as for `rope_halfsplit`), and k and v written to slot
    slots[t] of the cache: one launch.  A row with slot -1 is left out; of rows that name one slot the last one stays there."""
    dev = cache.device
    if ws.device != dev:
        raise _lib.AwqBackendError("rope_append: workspace and cache must be on one device")
    T = q.shape[0]
    qp, qr, qh = cache.rows(q, "q")
    H = q.shape[1]
    kp, kr, kh = cache.rows(k, "k", cache.n_kv_heads, T)
    vp, vr, vh = cache.rows(v, "v", cache.n_kv_heads, T)
    op, orow, oh = (qp, qr, qh) if q_out is None else cache.rows(q_out, "q_out", H, T)
    lut_p = _on(lut, "lut", torch.bfloat16, dev, 2)
    if lut.shape[1] != cache.head_dim or lut.shape[0] == 0:
        raise _lib.AwqBackendError(f"lut must be [positions, {cache.head_dim}], got {tuple(lut.shape)}")
    pos_p, slots_p = _on(positions, "positions", torch.int32, dev), _on(slots, "slots", torch.int32, dev)
    if positions.numel() != T or slots.numel() != T:
        _sizes(positions=(positions, T), slots=(slots, T))
    _call_on(dev, "awq_b200_rope_append", qp, qr, qh, kp, kr, kh, vp, vr, vh, lut_p, lut.shape[0], pos_p, slots_p, op, orow, oh, cache.ptr, T, H,
             ws.ptr, ws.nbytes)
    return q if q_out is None else q_out


def tree_attention(q, cache: KVCache, table, lens, q_start, ws: RequestWorkspace, mask=None, scale: Optional[float] = None, out=None):
    """out [T, n_heads, head_dim]: the step's rows q against their requests' cached tokens and the step's own (whose K and V
    are in the cache already: `rope_append`).  Row t of request r sees its lens[r] cached tokens and token j of the step if bit
    j of mask[t] (int64) is set, or without `mask` the tokens up to itself.  A row that sees nothing is 0.  Rows behind
    q_start[R] are left as they are in a given `out` (which may be q), 0 in a new one.  scale: head_dim ** -0.5 unless given."""
    dev = cache.device
    if ws.device != dev:
        raise _lib.AwqBackendError("tree_attention: workspace and cache must be on one device")
    qp, qr, qh = cache.rows(q, "q")
    T, H = q.shape[0], q.shape[1]
    if out is None:
        out = torch.zeros((T, H, cache.head_dim), dtype=cache.dtype, device=q.device)
    op, orow, oh = cache.rows(out, "out", H, T)
    R = lens.numel()
    lens_p, start_p = _on(lens, "lens", torch.int32, dev), _on(q_start, "q_start", torch.int32, dev)
    if q_start.numel() != R + 1:
        _sizes(q_start=(q_start, R + 1))
    table_p, stride, width = _table(table, R, dev)
    mask_p = None
    if mask is not None:
        mask_p = _on(mask, "mask", torch.int64, dev)
        if mask.numel() != T:
            _sizes(mask=(mask, T))
    _call_on(dev, "awq_b200_tree_attention", qp, qr, qh, cache.ptr, table_p, stride, width, lens_p, start_p, mask_p,
             cache.head_dim ** -0.5 if scale is None else float(scale), op, orow, oh, R, T, H, ws.ptr, ws.nbytes)
    return out


def page_keep(kv, table, lens, q_start, kept, free_pages, free_count, ws: RequestWorkspace, path=None, lens_out=None, free_count_out=None):
    """After a step: keep kept[r] of request r's tokens.  In every layer of kv [layers, 2, n_pages, page_size, n_kv_heads, head_dim] the
    rows path[q_start[r] + i] (indices in its tree, ascending; without `path` the first kept[r]) move to lens[r] + i; lens grows
    by kept and the pages behind it go back to `free_pages` (in place unless lens_out / free_count_out are given).
    kept[r] = -1 ends the request: length 0, all its pages free.  `path` has a place for every row of the step; a request with rows
    behind its end is left as it is, and ws.check() says so."""
    dev, R = ws.device, lens.numel()
    if kv.dim() != 6 or kv.shape[1] != 2 or kv.element_size() != 2 or kv.get_device() != dev or kv.numel() == 0:
        raise _lib.AwqBackendError(f"kv must be [layers, 2, n_pages, page_size, n_kv_heads, head_dim] of 16-bit values on cuda:{dev}, got "
                                   f"{tuple(kv.shape)} of {kv.dtype} on {kv.device}")
    shape, step = kv.shape, kv.stride()
    strides = [step[i] if shape[i] > 1 else 0 for i in range(5)]
    if step[5] != 1 or any(s % 8 or (s <= 0 and n > 1) for s, n in zip(strides, shape)):
        raise _lib.AwqBackendError("kv needs a unit stride over head_dim and positive multiples of 8 elsewhere")
    table_p, stride, width = _table(table, R, dev)
    lens_out = lens if lens_out is None else lens_out
    count_out = free_count if free_count_out is None else free_count_out
    i32 = torch.int32
    lens_p, lens_out_p, start_p, kept_p = (_on(lens, "lens", i32, dev), _on(lens_out, "lens_out", i32, dev), _on(q_start, "q_start", i32, dev),
                                           _on(kept, "kept", i32, dev))
    free_p, count_p, count_out_p = (_on(free_pages, "free_pages", i32, dev), _on(free_count, "free_count", i32, dev),
                                    _on(count_out, "free_count_out", i32, dev))
    if lens_out.numel() != R or q_start.numel() != R + 1 or kept.numel() != R or free_count.numel() != 1 or count_out.numel() != 1:
        _sizes(lens_out=(lens_out, R), q_start=(q_start, R + 1), kept=(kept, R), free_count=(free_count, 1), free_count_out=(count_out, 1))
    path_p, T = None, _lib.MAX_ROWS
    if path is not None:
        path_p, T = _on(path, "path", torch.int32, dev), path.numel()
    _call_on(dev, "awq_b200_page_keep", kv.data_ptr(), *strides, shape[0], *shape[2:], table_p, stride,
             width, lens_p, lens_out_p, start_p, kept_p, path_p, free_p, free_pages.numel(), count_p, count_out_p, R, T, ws.ptr, ws.nbytes)
    return lens_out


class LoraAdapters:
    """Low-rank adapters of one projection [K, N], resident: A bf16 [n, rank_max, K], B bf16 [n, N, rank_max] (the two matrices of
    each adapter as they are trained), scales f32 [n], ranks int32 [n] or None: how many rows of A and columns of B an
    adapter has; what lies behind them is not read."""

    def __init__(self, A: torch.Tensor, B: torch.Tensor, scales: torch.Tensor, ranks: Optional[torch.Tensor] = None):
        if not A.is_cuda or A.dim() != 3 or B.dim() != 3:
            raise _lib.AwqBackendError("LoraAdapters: A [n, rank_max, K] and B [n, N, rank_max] must be CUDA tensors")
        self.device = A.get_device()
        self.n, self.rank_max, self.K = A.shape
        self.N = B.shape[1]
        if tuple(B.shape) != (self.n, self.N, self.rank_max):
            raise _lib.AwqBackendError(f"LoraAdapters: B must be [{self.n}, N, {self.rank_max}], got {tuple(B.shape)}")
        if self.rank_max % 8 or not 0 < self.rank_max <= 128 or self.K % 8 or self.N % 8:
            raise _lib.AwqBackendError(f"LoraAdapters: rank_max must be a multiple of 8 up to 128, K and N multiples of 8, got {self.rank_max}, {self.K}, "
                                       f"{self.N}")
        self.A, self.B, self.scales, self.ranks = A, B, scales, ranks
        self._ptrs = (_on(A, "A", torch.bfloat16, self.device, 3), _on(B, "B", torch.bfloat16, self.device, 3),
                      _on(scales, "scales", torch.float32, self.device), None if ranks is None else _on(ranks, "ranks", torch.int32, self.device))
        _sizes(scales=(scales, self.n), **({} if ranks is None else dict(ranks=(ranks, self.n))))
        if not _aligned16(A, B):
            raise _lib.AwqBackendError("LoraAdapters: A and B must be 16-byte aligned")


def lora(x, adapters: LoraAdapters, idx, base, ws: RequestWorkspace, out=None, residual=None):
    """out bf16 [T, N] = bf16(base + scale (x A^T) B^T (+ residual)) with adapter idx[t] for row t of x bf16 [T, K], -1: none.  base is
    the shared projection's output, f32 sums (`gemv(..., f32_out=True)`) or bf16; out may be a bf16 base or the residual, not x."""
    dev = ws.device
    if adapters.device != dev:
        raise _lib.AwqBackendError("lora: workspace and adapters must be on one device")
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.get_device() != dev or x.shape[1] != adapters.K or x.stride(1) != 1:
        raise _lib.AwqBackendError(f"x must be bf16 [T, {adapters.K}] on cuda:{dev} with unit column stride, got {tuple(x.shape)} of {x.dtype} on {x.device}")
    T = x.shape[0]
    shape = (T, adapters.N)
    idx_p = _on(idx, "idx", torch.int32, dev)
    if idx.numel() != T:
        _sizes(idx=(idx, T))
    f32 = base.dtype == torch.float32
    base_p = _on(base, "base", torch.float32 if f32 else torch.bfloat16, dev, 2)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=x.device)
    out_p = _on(out, "out", torch.bfloat16, dev, 2)
    res_p = None if residual is None else _on(residual, "residual", torch.bfloat16, dev, 2)
    if base.shape != shape or out.shape != shape or (residual is not None and residual.shape != shape):
        raise _lib.AwqBackendError(f"base, out and residual must be {list(shape)}")
    _call_on(dev, "awq_b200_lora_bf16", x.data_ptr(), x.stride(0) if T > 1 else 0, *adapters._ptrs, adapters.n, adapters.rank_max, idx_p, base_p,
             1 if f32 else 0, res_p, out_p, T, adapters.K, adapters.N, ws.ptr, ws.nbytes)
    return out


def linear_bf16(x, W, out=None):
    """y [M, N] = x [M, K] @ W[N, K]^T with un-quantised bf16 weights (the bf16 sibling path)."""
    _want(x, torch.bfloat16, "x")
    _want(W, torch.bfloat16, "W")
    x2 = x.view(1, -1) if x.dim() == 1 else x
    if out is None:
        out = torch.empty((x2.shape[0], W.shape[0]), dtype=torch.bfloat16, device=x.device)
    ws = _parts("awq_b200_linear_workspace_bytes", out.device, x2.shape[0], x2.shape[1], W.shape[0])
    if ws is not None:
        _lib.call("awq_b200_linear_ws_bf16", _ptr(x2), _ptr(W), _ptr(out), x2.shape[0], x2.shape[1], W.shape[0], _ptr(ws), ws.numel(),
                  _stream())
        return out
    _lib.call("awq_b200_linear_bf16", _ptr(x2), _ptr(W), _ptr(out), x2.shape[0], x2.shape[1], W.shape[0], _stream())
    return out


def silu_mul(gate, up, out=None):
    """out = silu(gate) * up elementwise (bf16 in, f32 math, bf16 out)."""
    if out is None:
        out = torch.empty_like(gate)
    _lib.call("awq_b200_silu_mul_bf16", _ptr(_want(gate, torch.bfloat16, "gate")), _ptr(_want(up, torch.bfloat16, "up")),
              _ptr(out), gate.numel(), _stream())
    return out


def gemm_check():
    """Synchronise and raise if the tensor-core GEMM reported a device-side timeout."""
    _lib.call("awq_b200_gemm_check", _stream())


def repack_B_to_A(A_q, A_s, A_z, group_size=128) -> AwqWeight:
    """mlir-air logical layout (A_q u8 [M, K/2], A_s bf16 [G, M], A_z u8 [G, M]) -> layout A."""
    M, K = A_q.shape[0], A_q.shape[1] * 2
    G = K // group_size
    dev = A_q.device
    qw = torch.empty((K, M // 8), dtype=torch.int32, device=dev)
    qz = torch.empty((G, M // 8), dtype=torch.int32, device=dev)
    sc = torch.empty((G, M), dtype=torch.bfloat16, device=dev)
    _lib.call("awq_b200_repack_B_to_A", _ptr(_want(A_q, torch.uint8, "A_q")), _ptr(_want(A_s, torch.bfloat16, "A_s")),
              _ptr(_want(A_z, torch.uint8, "A_z")), _ptr(qw), _ptr(qz), _ptr(sc), M, K, group_size, _stream())
    return AwqWeight(qw, qz, sc, group_size)


def repack_A_to_B(w: AwqWeight):
    M, K, G = w.N, w.K, w.K // w.group_size
    dev = w.qweight.device
    A_q = torch.empty((M, K // 2), dtype=torch.uint8, device=dev)
    A_s = torch.empty((G, M), dtype=torch.bfloat16, device=dev)
    A_z = torch.empty((G, M), dtype=torch.uint8, device=dev)
    _lib.call("awq_b200_repack_A_to_B", _ptr(w.qweight), _ptr(w.qzeros), _ptr(w.scales), _ptr(A_q), _ptr(A_s),
              _ptr(A_z), M, K, w.group_size, _stream())
    return A_q, A_s, A_z


def repack_C_to_B(packed, M: int, K: int, group_size=128, m_tile=8, k_chunk=2048):
    """Per-tile packed buffer (uint8, tiles in (row block, k chunk) order: the reference's NPU layout
    for the GEMV and, with M = N and m_tile = N_TILE, for the GEMM) -> layout B on the device."""
    _want(packed, torch.uint8, "packed")
    G = K // group_size
    tile = m_tile * (k_chunk // 2) + 3 * (k_chunk // group_size) * m_tile
    if packed.numel() != (M // m_tile) * (K // k_chunk) * tile:
        raise _lib.AwqBackendError(f"packed buffer has {packed.numel()} bytes, expected {(M // m_tile) * (K // k_chunk)} "
                                   f"tiles of {tile}")
    dev = packed.device
    A_q = torch.empty((M, K // 2), dtype=torch.uint8, device=dev)
    A_s = torch.empty((G, M), dtype=torch.bfloat16, device=dev)
    A_z = torch.empty((G, M), dtype=torch.uint8, device=dev)
    _lib.call("awq_b200_repack_C_to_B", _ptr(packed), _ptr(A_q), _ptr(A_s), _ptr(A_z), M, K, group_size, m_tile, k_chunk,
              _stream())
    return A_q, A_s, A_z


def repack_C_to_A(packed, M: int, K: int, group_size=128, m_tile=8, k_chunk=2048) -> AwqWeight:
    """Per-tile packed buffer -> resident layout-A weight (two device passes, once per weight)."""
    return repack_B_to_A(*repack_C_to_B(packed, M, K, group_size, m_tile, k_chunk), group_size)
