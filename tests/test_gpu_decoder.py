"""Decoder layers of many requests over a paged cache: prompts, drafted trees, accepted paths and adapters, against a plain decoder that keeps
every request's tokens in lists."""
import random

import numpy as np
import pytest
import torch

from request_util import i32, starts

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
H, HEADS, KV, D, INTER, PAGE = 512, 8, 2, 64, 1024, 16


def make(layers=2, adapters=True, seed=0):
    from gpu_util import dev_weight, synth_awq
    from mlir_air_b200 import ops
    from mlir_air_b200.decoder import DecoderLayer, DecoderStack, PagedKVCache
    from mlir_air_b200.ffn import FFNLayer
    from mlir_air_b200.programming_examples.llms.llama32_1b_int4.multi_launch_builder.rms_qkv_int4_rope_multi import generate_rope_lut
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i in range(layers):
        # nibbles about the zero point 8 and small scales: activations stay of order one through the layers
        w = lambda K, N, s: dev_weight(*synth_awq(K, N, seed=seed + 10 * i + s, scale_lo=0.002, scale_hi=0.006))  # noqa: B023, E731
        gamma = lambda: (torch.rand(H, device="cuda", generator=gen) * 0.2 + 0.9).to(BF)  # noqa: E731
        ad = lambda K, N: ops.LoraAdapters(  # noqa: E731
            (torch.randn((3, 16, K), device="cuda", generator=gen) * K ** -0.5).to(BF), (torch.randn((3, N, 16), device="cuda", generator=gen) * 0.3).to(BF),
            torch.tensor([1.0, 0.5, 2.0], device="cuda"), i32([16, 5, 9])) if adapters else None
        N = (HEADS + 2 * KV) * D
        out.append(DecoderLayer(w(H, N, 1), w(HEADS * D, H, 2), gamma(), FFNLayer(ops.interleave_gate_up(w(H, INTER, 3), w(H, INTER, 4)), w(INTER, H, 5), gamma()),
                                ad(H, N), ad(HEADS * D, H)))
    lut = torch.from_numpy(np.asarray(generate_rope_lut(D, seq_len=400), dtype=np.float32)).to(BF).cuda()
    cache = PagedKVCache(layers, 120, PAGE, KV, D, requests=4, max_tokens=400)
    return DecoderStack(out, cache, HEADS, lut)


class Plain:
    """The same decoder in 64 bits, request by request, rounded to bf16 where the framework's path hands over bf16."""

    def __init__(self, stack):
        from mlir_air_b200 import ops

        def wide(w):  # (q - z) s, not rounded
            return ops.dequant(ops.AwqWeight(w.qweight, w.qzeros, torch.ones_like(w.scales))).double() * w.scales.double().repeat_interleave(128, 0)
        self.s = stack
        self.w = [dict(qkv=wide(l.qkv), o=wide(l.o), gu=wide(l.ffn.gateup), down=wide(l.ffn.down)) for l in stack.layers]
        self.cache = [[(torch.zeros((0, KV, D), dtype=torch.float64, device="cuda"),) * 2 for _ in range(4)] for _ in stack.layers]

    def norm(self, x, gamma):
        return (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + self.s.eps) * gamma.double()).to(BF).double()

    def project(self, x, w, ad, idx, residual=None):
        y = x @ w
        for t, a in enumerate(idx):
            if ad is not None and a >= 0:
                r = int(ad.ranks[a])
                y[t] += float(ad.scales[a]) * (ad.B[a, :, :r].double() @ (ad.A[a, :r].double() @ x[t]))
        return (y if residual is None else y + residual).to(BF).double()

    def step(self, h, lens, new, parents, idx):
        """Hidden states behind the last layer, and every layer's new K and V."""
        h, st, fresh = h.double(), starts(new), []
        seen, depth = [], []
        for r, n in enumerate(new):
            for j in range(n):
                chain, p = [j], j
                while parents is not None and parents[st[r] + p] >= 0:
                    p = parents[st[r] + p]
                    chain.append(p)
                seen.append(sorted(chain) if parents is not None else list(range(j + 1)))
                depth.append(lens[r] + (len(chain) - 1 if parents is not None else j))
        turn = self.s.lut[torch.tensor(depth, device="cuda")].double()
        for i, (l, w) in enumerate(zip(self.s.layers, self.w)):
            qkv = self.project(self.norm(h, l.gamma), w["qkv"], l.qkv_lora, idx)
            q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([HEADS * D, KV * D, KV * D], 1))

            def rotate(x):
                a, b, c, s = x[..., :D // 2], x[..., D // 2:], turn[:, None, :D // 2], turn[:, None, D // 2:]
                return torch.cat([a * c - b * s, a * s + b * c], -1).to(BF).double()
            q, k = rotate(q), rotate(k)
            fresh.append((k, v))
            a = torch.zeros_like(q)
            for r, n in enumerate(new):
                for j in range(n):
                    pick = [st[r] + x for x in seen[st[r] + j]]
                    ks, vs = torch.cat([self.cache[i][r][0], k[pick]]), torch.cat([self.cache[i][r][1], v[pick]])
                    for hd in range(HEADS):
                        g = hd * KV // HEADS
                        a[st[r] + j, hd] = torch.softmax(ks[:, g] @ q[st[r] + j, hd] * D ** -0.5, 0) @ vs[:, g]
            h = self.project(a.to(BF).double().flatten(1), w["o"], l.o_lora, idx, h)
            gu = (self.norm(h, l.ffn.gamma) @ w["gu"]).to(BF).double()
            inter = (torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]).to(BF).double()
            h = (inter @ w["down"] + h).to(BF).double()
        return h, fresh

    def keep(self, fresh, new, kept, path):
        st = starts(new)
        for i, (k, v) in enumerate(fresh):
            for r in range(len(new)):
                if kept[r] < 0:
                    self.cache[i][r] = (k[:0], v[:0])
                    continue
                pick = [st[r] + p for p in (path[st[r]:st[r] + kept[r]] if path is not None else range(kept[r]))]
                self.cache[i][r] = tuple(torch.cat([c, x[pick]]) for c, x in zip(self.cache[i][r], (k, v)))


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("adapters", [True, False])
def test_prompts_trees_and_single_tokens(adapters):
    """The bound is the framework's own for its int4 blocks, rel-L2 1e-2, here behind two whole layers; the plain decoder rounds where the
    kernels do, so that only their sums' order and a few roundings more (f16 between an FFN's kernels) lie between the two."""
    stack = make(adapters=adapters)
    plain = Plain(stack)
    rng = random.Random(3)
    R, lens = 4, [0] * 4
    for step, kind in enumerate(["prompt", "tree", "one", "tree", "prompt", "one", "tree"]):
        if kind == "prompt":
            new = [rng.randint(5, 60) if l == 0 else 1 for l in lens]
        else:
            new = [rng.randint(2, 12) if kind == "tree" else 1 for _ in lens]
        T, st = sum(new), starts(new)
        parents = [rng.randint(max(-1, j - 3), j - 1) for n in new for j in range(n)] if kind == "tree" else None
        plan = stack.cache.plan(i32(new), T, parents=None if parents is None else i32(parents))
        h = torch.randn((T, H), device="cuda").to(BF)
        idx = [(r % 4) - 1 for r, n in enumerate(new) for _ in range(n)]
        got = stack.step(h, plan, i32(idx) if adapters else None)
        stack.check()
        want, fresh = plain.step(h, lens, new, parents, idx if adapters else [-1] * T)
        assert rel(got, want) <= 1e-2, (step, kind, rel(got, want))
        # accept part of the trees, everything else whole; one request ends half way
        kept = [rng.randint(1, n) if kind == "tree" else n for n in new]
        path = [x for n, k in zip(new, kept) for x in sorted(rng.sample(range(n), k)) + [0] * (n - k)] if kind == "tree" else None
        if step == 3:
            kept[1] = -1
        stack.cache.keep(plan, i32(kept), None if path is None else i32(path))
        stack.check()
        plain.keep(fresh, new, kept, path)
        lens = [0 if k < 0 else l + k for l, k in zip(lens, kept)]
        assert stack.cache.lens.tolist() == lens
    held = sum(-(-l // PAGE) for l in lens)
    assert int(stack.cache.free_count) == 120 - held


def test_a_captured_step_serves_later_ones():
    """Plan, layers and keep of one-token steps in one graph, replayed: the same hidden states and cache as eager steps."""
    eager, graphed = make(), make()
    new, kept, idx = i32([1] * 4), i32([1] * 4), i32([0, -1, 2, 1])
    h = torch.zeros((4, H), dtype=BF, device="cuda")

    def prompt(stack):
        gen = torch.Generator(device="cuda").manual_seed(1)
        n = [20, 31, 5, 16]
        plan = stack.cache.plan(i32(n), sum(n))
        stack.step(torch.randn((sum(n), H), device="cuda", generator=gen).to(BF), plan, i32([0] * sum(n)))
        stack.cache.keep(plan, i32(n))

    def one(stack):
        plan = stack.cache.plan(new, 4)
        out = stack.step(h, plan, idx)
        stack.cache.keep(plan, kept)
        return out
    prompt(eager)
    prompt(graphed)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    state = [t.clone() for t in (graphed.cache.lens, graphed.cache.table, graphed.cache.free_count)]
    with torch.cuda.stream(side):
        one(graphed)  # warm-up; its step is taken back
    torch.cuda.current_stream().wait_stream(side)
    for t, s in zip((graphed.cache.lens, graphed.cache.table, graphed.cache.free_count), state):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one(graphed)
    gen = torch.Generator(device="cuda").manual_seed(2)
    for _ in range(20):
        h.copy_(torch.randn((4, H), device="cuda", generator=gen).to(BF))
        want = one(eager)
        graph.replay()
        assert torch.equal(out, want)
    eager.check()
    graphed.check()
    assert torch.equal(eager.cache.lens, graphed.cache.lens) and graphed.cache.lens.tolist() == [40, 51, 25, 36]


def test_weights_that_do_not_fit_are_refused():
    from mlir_air_b200._lib import AwqBackendError
    from mlir_air_b200.decoder import DecoderStack
    stack = make()
    with pytest.raises(AwqBackendError):
        DecoderStack(stack.layers[:1], stack.cache, HEADS, stack.lut)
    with pytest.raises(AwqBackendError):
        DecoderStack(stack.layers, stack.cache, HEADS * 2, stack.lut)
    plan = stack.cache.plan(i32([1, 1, 0, 0]), 2)
    with pytest.raises(AwqBackendError):
        stack.step(torch.zeros((3, H), dtype=BF, device="cuda"), plan)
    stack.check()


def test_a_step_without_pages_is_reported():
    from mlir_air_b200._lib import AwqBackendError
    stack = make()
    stack.cache.plan(i32([399] * 4), 1600)
    stack.check()
    stack.cache.plan(i32([400] * 4), 1600)  # (nothing was kept: the same requests again, from 20 pages)
    with pytest.raises(AwqBackendError, match="not enough free pages"):
        stack.check()
