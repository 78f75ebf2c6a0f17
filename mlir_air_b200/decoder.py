"""Whole decoder layers of many requests on int4 weights: the attention half around a paged cache, and the FFN.

The reference's decode loop runs, per token and layer, the QKV block, attention on the host and the block behind it
(llms/llama32_1b_int4/llama32_1b_int4_decode.py:176-313), for one request.  Here a step takes the new tokens of all
requests at once (one each, drafted trees, prompts), and nothing comes back to the host between the layers:

    plan   = cache.plan(new, T)                 pages, slots, positions, masks            (one launch per step)
    per layer
      qkv  = rmsnorm(h, gamma) . W_qkv  (+ adapters)
      q    = RoPE(q); K and V into the cache     (one launch)
      a    = attention of q over the pages
      h    = h + a . W_o  (+ adapters)
      h    = h + down(swiglu(gateup . rmsnorm(h, gamma_ffn)))
    cache.keep(plan, kept, path)                 accepted tokens stay, pages behind them go back
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import ops
from ._lib import AwqBackendError
from .ffn import FFNLayer
from .ops import AwqWeight, KVCache, LoraAdapters, RequestWorkspace, StepPlan


class PagedKVCache:
    """K and V of all layers in pages, and the requests that live in them: block tables, lengths, the free pages.

    `requests` slots for requests of up to `max_tokens` each share `n_pages` pages of `page_size` tokens.  A slot starts empty
    (length 0) and is empty again once `keep` was given -1 for it."""

    def __init__(self, layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, requests: int, max_tokens: int,
                 dtype=torch.bfloat16, device="cuda"):
        i32 = dict(dtype=torch.int32, device=device)
        self.page_size = page_size
        # zeros: pages are read in whole tiles, and a fresh page should not hold what an allocator left there
        self.kv = torch.zeros((layers, 2, n_pages, page_size, n_kv_heads, head_dim), dtype=dtype, device=device)
        self.layers = [KVCache(self.kv[i, 0], self.kv[i, 1]) for i in range(layers)]
        self.table = torch.full((requests, -(-max_tokens // page_size)), -1, **i32)
        self.lens = torch.zeros(requests, **i32)
        self.free_pages = torch.arange(n_pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), n_pages, **i32)
        self.ws = RequestWorkspace(device)

    def plan(self, new: torch.Tensor, T: int, parents: Optional[torch.Tensor] = None, out: Optional[StepPlan] = None) -> StepPlan:
        """Pages and rows of a step that brings new[r] tokens of every request; see ops.page_plan."""
        return ops.page_plan(self.lens, new, self.table, self.free_pages, self.free_count, self.page_size, T, self.ws, parents=parents, out=out)

    def append(self, layer: int, q, k, v, lut, plan: StepPlan, q_out=None):
        return ops.rope_append(q, k, v, lut, plan.positions, plan.slots, self.layers[layer], self.ws, q_out=q_out)

    def attend(self, layer: int, q, plan: StepPlan, out=None):
        return ops.tree_attention(q, self.layers[layer], self.table, self.lens, plan.q_start, self.ws, mask=plan.mask, out=out)

    def keep(self, plan: StepPlan, kept: torch.Tensor, path: Optional[torch.Tensor] = None):
        """The step's accepted tokens stay (kept[r] of request r, -1: the request ends); see ops.page_keep."""
        return ops.page_keep(self.kv, self.table, self.lens, plan.q_start, kept, self.free_pages, self.free_count, self.ws, path=path)

    def check(self):
        """Synchronise and raise if a step since the last check did not fit."""
        self.ws.check()


@dataclass
class DecoderLayer:
    """One layer's resident weights: qkv [H, (n_heads + 2 n_kv_heads) head_dim] (Wq | Wk | Wv), o [n_heads head_dim, H], the norm in front of the
    attention, the FFN (with its norm weight), and adapters of many requests beside the two projections."""
    qkv: AwqWeight
    o: AwqWeight
    gamma: torch.Tensor
    ffn: FFNLayer
    qkv_lora: Optional[LoraAdapters] = None
    o_lora: Optional[LoraAdapters] = None


class DecoderStack:
    """A stack of decoder layers over a PagedKVCache.  step(h, plan) takes the hidden states of the plan's rows [T, H] and returns
    those behind the last layer; every launch goes to the current stream, so a step can be captured into a graph."""

    MAX_DECODE_ROWS = 64  # rows of the decode kernels; more go through the prefill GEMM

    def __init__(self, layers: Sequence[DecoderLayer], cache: PagedKVCache, n_heads: int, lut: torch.Tensor, eps: float = 1e-5):
        """lut: bf16 [positions, head_dim], rows [cos | sin] (rms_qkv_int4_rope_multi.generate_rope_lut)."""
        self.layers, self.cache, self.lut, self.eps = list(layers), cache, lut, eps
        self.n_heads, self.n_kv, self.head_dim = n_heads, cache.layers[0].n_kv_heads, cache.layers[0].head_dim
        self.hidden = self.layers[0].qkv.K
        q_cols, kv_cols = n_heads * self.head_dim, self.n_kv * self.head_dim
        if len(self.layers) != len(cache.layers):
            raise AwqBackendError(f"{len(self.layers)} layers over a cache of {len(cache.layers)}")
        for l in self.layers:
            if (l.qkv.K, l.qkv.N, l.o.K, l.o.N) != (self.hidden, q_cols + 2 * kv_cols, q_cols, self.hidden) or l.ffn.gamma is None or \
                    (l.ffn.gateup.K, l.ffn.gateup.N, l.ffn.down.N) != (self.hidden, 2 * l.ffn.down.K, self.hidden):
                raise AwqBackendError(f"a layer's weights do not fit {n_heads} / {self.n_kv} heads of {self.head_dim} and {self.hidden} hidden values")
            for ad, w in ((l.qkv_lora, l.qkv), (l.o_lora, l.o)):
                if ad is not None and (ad.K, ad.N) != (w.K, w.N):
                    raise AwqBackendError(f"adapters of [{ad.K}, {ad.N}] beside a projection of [{w.K}, {w.N}]")
        widest = max(max(l.qkv.N, l.ffn.gateup.N) for l in self.layers)
        deepest = max(max(l.o.K, l.ffn.down.K, self.hidden) for l in self.layers)
        device = self.layers[0].gamma.device
        self.ws = ops.Workspace(deepest, widest, device=device)
        self.gemm_ws = ops.GemmDecodeWorkspace(widest, device=device, batch=self.MAX_DECODE_ROWS, K=deepest)

    def _project(self, x, w: AwqWeight, adapters, idx, residual=None):
        """bf16(x W (+ adapters) (+ residual)): one rounding on the decode path, where the adapters take the projection's f32 sums; more rows go
        through the prefill GEMM, which rounds the weights to bf16, and adapters are added to its bf16 output."""
        if x.shape[0] > self.MAX_DECODE_ROWS:
            if adapters is None or idx is None:
                return ops.gemm(x, w, residual=residual)
            return ops.lora(x, adapters, idx, ops.gemm(x, w), self.cache.ws, residual=residual)
        if adapters is None or idx is None:
            return ops.gemv(x, w, self.ws, residual=residual)
        return ops.lora(x, adapters, idx, ops.gemv(x, w, self.ws, f32_out=True), self.cache.ws, residual=residual)

    def _ffn(self, h, l: FFNLayer):
        B = h.shape[0]
        if B > self.MAX_DECODE_ROWS:
            return ops.gemm(ops.gemm(ops.rmsnorm(h, l.gamma, self.eps), l.gateup, swiglu=True), l.down, residual=h)
        if B > 8 and self.gemm_ws.fits_layer(B, self.hidden, l.down.K):
            return ops.ffn_layer_decode(h, l.gateup, l.down, self.gemm_ws, l.gamma, self.eps)
        return ops.ffn_decode(h, l.gateup, l.down, self.ws, gamma=l.gamma, eps=self.eps, residual=h)

    def step(self, h: torch.Tensor, plan: StepPlan, adapter: Optional[torch.Tensor] = None) -> torch.Tensor:
        """h bf16 [T, H] -> bf16 [T, H].  adapter: int32 [T], each row's adapter (-1: none) in every layer that has some."""
        T = plan.slots.numel()
        if tuple(h.shape) != (T, self.hidden):
            raise AwqBackendError(f"h must be [{T}, {self.hidden}], got {tuple(h.shape)}")
        if T == 0:
            return h
        q_cols, kv_cols = self.n_heads * self.head_dim, self.n_kv * self.head_dim
        for i, l in enumerate(self.layers):
            qkv = self._project(ops.rmsnorm(h, l.gamma, self.eps), l.qkv, l.qkv_lora, adapter)
            q, k, v = (t.unflatten(1, (-1, self.head_dim)) for t in qkv.split([q_cols, kv_cols, kv_cols], 1))
            self.cache.append(i, q, k, v, self.lut, plan)
            a = self.cache.attend(i, q, plan)
            h = self._project(a.view(T, q_cols), l.o, l.o_lora, adapter, residual=h)
            h = self._ffn(h, l.ffn)
        return h

    def check(self):
        """Synchronise and raise if a step did not fit or a device-side wait gave up."""
        self.cache.check()
        self.ws.check()
