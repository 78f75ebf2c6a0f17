"""Decoder layers of many requests against a plain decoder that rounds where each size of a step does, step by step from the same cache.

What the path rounds depends on the rows of a step.  Up to 64 rows a projection takes its weights as they are, and the adapters and the residual
its f32 sums: one rounding.  More rows go through the prefill GEMM, whose weights are rounded to bf16 once they are dequantised, and whose
output is bf16 before adapters are added.  An FFN's intermediates are bf16 there and from 9 to 32 rows, else fp16."""
import random

import pytest
import torch

from request_util import i32, starts
from test_gpu_decoder import BF, D, H, HEADS, INTER, KV, PAGE, Plain, make, rel

pytestmark = pytest.mark.gpu


class PathPlain(Plain):
    """In 64 bits, rounded as the step's size has it; every step starts from the tokens that the stack's own cache holds."""

    def __init__(self, stack):
        super().__init__(stack)
        self.rounded = [{k: w.to(BF).double() for k, w in l.items()} for l in self.w]
        self.exact = self.w

    def project(self, x, w, ad, idx, residual=None):
        if x.shape[0] <= 64:
            return super().project(x, w, ad, idx, residual)
        y = x @ w
        if any(a >= 0 for a in idx):
            y = super().project(x, w, None, idx)
            for t, a in enumerate(idx):
                if a >= 0:
                    r = int(ad.ranks[a])
                    y[t] += float(ad.scales[a]) * (ad.B[a, :, :r].double() @ (ad.A[a, :r].double() @ x[t]))
        return (y if residual is None else y + residual).to(BF).double()

    def ffn(self, h, l, w):
        T = h.shape[0]
        t = BF if T > 64 or 8 < T <= 32 and self.s.gemm_ws.fits_layer(T, H, INTER) else torch.float16
        x = (h * torch.rsqrt((h * h).mean(-1, keepdim=True) + self.s.eps) * l.ffn.gamma.double()).to(t).double()
        gu = x @ w["gu"]
        inter = (torch.nn.functional.silu(gu[:, 0::2]) * gu[:, 1::2]).to(t).double()
        return (inter @ w["down"] + h).to(BF).double()

    def step(self, h, lens, new, parents, idx):
        table, cache = self.s.cache.table.long(), self.s.cache.kv.double()
        h, st = h.double(), starts(new)
        weights = self.rounded if h.shape[0] > 64 else self.exact
        seen, depth = [], []
        for r, n in enumerate(new):
            for j in range(n):
                chain = [j]
                while parents is not None and parents[st[r] + chain[-1]] >= 0:
                    chain.append(parents[st[r] + chain[-1]])
                seen.append(sorted(chain) if parents is not None else list(range(j + 1)))
                depth.append(lens[r] + (len(chain) - 1 if parents is not None else j))
        turn = self.s.lut[torch.tensor(depth, device="cuda")].double()[:, None]
        for i, (l, w) in enumerate(zip(self.s.layers, weights)):
            qkv = self.project(self.norm(h, l.gamma), w["qkv"], l.qkv_lora, idx)
            q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([HEADS * D, KV * D, KV * D], 1))
            c, s = turn[..., :D // 2], turn[..., D // 2:]
            q, k = (torch.cat([x[..., :D // 2] * c - x[..., D // 2:] * s, x[..., :D // 2] * s + x[..., D // 2:] * c], -1).to(BF).double() for x in (q, k))
            a = torch.zeros_like(q)
            for r, n in enumerate(new):
                p = torch.arange(lens[r], device="cuda")
                old = cache[i][:, table[r, p // PAGE], p % PAGE]  # [2, tokens, KV, D]
                for j in range(n):
                    pick = [st[r] + x for x in seen[st[r] + j]]
                    ks, vs = (torch.cat([o, x[pick]]).repeat_interleave(HEADS // KV, 1) for o, x in zip(old, (k, v)))
                    a[st[r] + j] = torch.einsum("ph,phd->hd", torch.softmax(torch.einsum("phd,hd->ph", ks, q[st[r] + j]) * D ** -0.5, 0), vs)
            h = self.project(a.to(BF).double().flatten(1), w["o"], l.o_lora, idx, h)
            h = self.ffn(h, l, w)
        return h


@pytest.mark.parametrize("adapters", [True, False])
@pytest.mark.parametrize("seed", range(6))
def test_steps_from_one_cache(seed, adapters):
    """The bound is the framework's for its int4 blocks, rel-L2 1e-2, here behind two whole layers.  Between the two lie the order of f32 sums and
    attention's 16-bit weights, and the roundings that these turn over: on a restatement of both sides on the host, 7.4e-3 at most in 200 draws."""
    stack = make(adapters=adapters, seed=100 * seed)
    plain = PathPlain(stack)
    rng, gen = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
    lens = [0] * 4
    for step, kind in enumerate(["prompt", "tree", "one", "tree", "prompt", "one", "tree"]):
        if kind == "prompt":
            new = [rng.randint(5, 60) if n == 0 else rng.randint(1, 20) for n in lens]
        else:
            new = [rng.randint(2, 12) if kind == "tree" else 1 for _ in lens]
        T, st = sum(new), starts(new)
        parents = [rng.randint(max(-1, j - 3), j - 1) for n in new for j in range(n)] if kind == "tree" else None
        plan = stack.cache.plan(i32(new), T, parents=None if parents is None else i32(parents))
        h = torch.randn((T, H), device="cuda", generator=gen).to(BF)
        idx = [(r % 4) - 1 for r, n in enumerate(new) for _ in range(n)] if adapters else [-1] * T
        want = plain.step(h, lens, new, parents, idx)
        got = stack.step(h, plan, i32(idx) if adapters else None)
        stack.check()
        assert rel(got, want) <= 1e-2, (step, kind, T, rel(got, want))
        kept = [rng.randint(1, n) if kind == "tree" else n for n in new]
        path = [x for n, k in zip(new, kept) for x in sorted(rng.sample(range(n), k)) + [0] * (n - k)] if kind == "tree" else None
        if step == 3:
            kept[1] = -1
        stack.cache.keep(plan, i32(kept), None if path is None else i32(path))
        stack.check()
        lens = [0 if k < 0 else n + k for n, k in zip(lens, kept)]
        assert stack.cache.lens.tolist() == lens
