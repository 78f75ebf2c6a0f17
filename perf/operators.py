"""One decode step of many requests around the int4 projections: paged cache, drafted tokens, adapters.

A case is a dict of plain values; `op` says which operator it is:

  plan    page_plan: block tables, slots, positions and ancestor masks of a step, from the requests' lengths
  append  rope_append: RoPE of Q and K, and K and V into their cache slots
  attend  tree_attention: the drafted tokens of every request against its cached tokens and their own ancestors
  keep    page_keep: the accepted tokens' cache rows moved together, lengths and free pages brought up to date
  lora    lora: each row's low-rank adapter added to a shared projection's output

`run` computes them in elementary torch operations (f32, one rounding at the end), or, where `own` is set, calls the framework.
Request lengths follow from the case alone, the values, page orders, trees and (for the plan) lengths from the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # Interactive decoding: four requests, one token each.  All latency.
        dict(name="plan_b4", op="plan", requests=4, new_lo=1, new_hi=1, len_hi=2000, page=16, tree=False),
        # A full server: 512 requests with drafted trees of 2 to 32 tokens.
        dict(name="plan_b512_trees", op="plan", requests=512, new_lo=2, new_hi=32, len_hi=16000, page=16, tree=True),
        # One token of the 1B model (32 heads of 64, 8 KV heads).
        dict(name="append_1b_b1", op="append", requests=1, new_lo=1, new_hi=1, heads=32, kv=8, dim=64, page=16, len_hi=500, dtype="bf16"),
        # Eight prompts of ragged lengths at once, Llama-3-8B heads.
        dict(name="append_8b_prompts", op="append", requests=8, new_lo=333, new_hi=1999, heads=32, kv=8, dim=128, page=64, len_hi=100,
             dtype="bf16"),
        # One token of the 1B model against a short conversation: latency.
        dict(name="attend_1b_b1", op="attend", requests=1, new_lo=1, new_hi=1, len_lo=777, len_hi=777, heads=32, kv=8, dim=64, page=16,
             tree=False, dtype="bf16"),
        # Trees of 8 to 32 drafted tokens of 16 requests, Llama-3-8B heads, conversations of ragged lengths.
        dict(name="attend_8b_trees", op="attend", requests=16, new_lo=8, new_hi=32, len_lo=300, len_hi=6000, heads=32, kv=8, dim=128,
             page=16, tree=True, dtype="bf16"),
        # 64 requests, one token each, long conversations, Llama-3-70B heads: the cache's bytes.
        dict(name="attend_70b_b64", op="attend", requests=64, new_lo=1, new_hi=1, len_lo=1000, len_hi=16000, heads=64, kv=8, dim=128,
             page=64, tree=False, dtype="bf16"),
        # Two requests with trees of 64 tokens over long documents, Llama-3-70B heads: the tensor cores' case.
        dict(name="attend_70b_trees_long", op="attend", requests=2, new_lo=64, new_hi=64, len_lo=32000, len_hi=32000, heads=64, kv=8,
             dim=128, page=64, tree=True, dtype="bf16"),
        # One request accepts a few of eight drafted tokens, 16 layers of the 1B model.
        dict(name="keep_1b_b1", op="keep", requests=1, new_lo=8, new_hi=8, len_hi=60, kept=3, layers=16, kv=8, dim=64, page=16,
             dtype="bf16"),
        # 32 requests accept 5 of up to 32 drafted tokens, 8 layers of Llama-3-8B.
        dict(name="keep_8b_b32", op="keep", requests=32, new_lo=6, new_hi=32, len_hi=90, kept=5, layers=8, kv=8, dim=128, page=16,
             dtype="bf16"),
        # Four requests with adapters of their own beside a square projection of the 1B model, one token each, on its f32 sums.
        dict(name="lora_1b_b4", op="lora", requests=4, new_lo=1, new_hi=1, K=2048, N=2048, adapters=8, rank_max=16, rank_lo=16,
             base="f32"),
        # Nine prompts of ragged lengths on seven adapters of mixed ranks beside Llama-3-8B's up projection.
        dict(name="lora_8b_prompts", op="lora", requests=9, new_lo=100, new_hi=700, K=4096, N=14336, adapters=7, rank_max=64, rank_lo=8,
             base="bf16"),
    ]


def _log_int(rng, lo, hi, step=1):
    """A whole multiple of `step` in [lo, hi], spread over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(max(int(round(v / step)) * step, -(-lo // step) * step), hi // step * step)


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "keep", "lora", "lora"])
    page = rng.choice([8, 16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv, dim = rng.choice([1, 2, 4, 8, 8, 12]), rng.choice([64, 128])
    if op == "plan":
        tree = rng.random() < 0.6
        hi = _log_int(rng, 1, 64) if tree else _log_int(rng, 1, 500)
        return dict(op=op, requests=_log_int(rng, 1, min(1024, 32768 // hi)), new_lo=rng.randint(0, hi), new_hi=hi,
                    len_hi=_log_int(rng, 10, 32000), page=page, tree=tree)
    if op == "append":
        hi = _log_int(rng, 1, 2000)
        return dict(op=op, requests=_log_int(rng, 1, max(1, min(256, 8000 // hi))), new_lo=rng.randint(1, hi), new_hi=hi,
                    heads=kv * rng.choice([1, 2, 3, 4, 8]), kv=kv, dim=dim, page=page, len_hi=_log_int(rng, 10, 500), dtype=dtype)
    if op == "attend":
        while True:
            hi = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 2, 64), _log_int(rng, 65, 512)])
            c = dict(op=op, requests=_log_int(rng, 1, 128), new_lo=rng.randint(1, hi), new_hi=hi,
                     len_lo=rng.choice([0, _log_int(rng, 1, 2000), _log_int(rng, 1, 2000)]), heads=kv * rng.choice([1, 2, 3, 4, 5, 8]),
                     kv=kv, dim=dim, page=page, tree=1 < hi <= 64 and rng.random() < 0.7, dtype=dtype)
            c["len_hi"] = _log_int(rng, max(c["len_lo"], 1), 32000)
            w = work(c)
            # (the padded scores and gathered keys of the plain form have to fit as well)
            if w["flops"] <= 1.3e11 and w["bytes"] <= 1.5e9 and c["requests"] * c["len_hi"] * max(kv * dim, c["heads"] * hi) <= 1.2e9:
                return c
    if op == "keep":
        hi = _log_int(rng, 2, 64)
        requests = _log_int(rng, 1, 48)
        return dict(op=op, requests=requests, new_lo=rng.randint(1, hi), new_hi=hi, len_hi=_log_int(rng, 5, 90), kept=rng.randint(1, 8),
                    layers=rng.choice([1, 2, 5, 8]), kv=kv, dim=dim, page=min(page, 32), dtype=dtype)
    while True:
        hi = _log_int(rng, 1, 700)
        c = dict(op=op, requests=_log_int(rng, 1, 64), new_lo=rng.randint(1, hi), new_hi=hi, K=_log_int(rng, 512, 16384, 8),
                 N=_log_int(rng, 512, 28672, 8), adapters=_log_int(rng, 1, 64), rank_max=rng.choice([8, 16, 32, 64, 128]),
                 base=rng.choice(["f32", "bf16"]))
        c["rank_lo"] = rng.randint(1, c["rank_max"])
        w = work(c)
        if w["flops"] <= 7e9 and w["bytes"] <= 1.5e8 and c["adapters"] * c["rank_max"] * (c["K"] + c["N"]) <= 1.5e8:
            return c


def _spread(n, lo, hi, tag):
    """n whole numbers from lo to hi, spread over their logarithm in a ragged order that follows from the arguments alone."""
    rng = random.Random("%s %d %d %d" % (tag, n, lo, hi))
    return [int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1 if i else hi for i in range(n)]


def _new(case):
    return _spread(case["requests"], case["new_lo"], case["new_hi"], "new")


def _lens(case):
    return _spread(case["requests"], case.get("len_lo", 1), case["len_hi"], "len")


def _ranks(case):
    return _spread(case["adapters"], case["rank_lo"], case["rank_max"], "rank")


def _adapter_of(case):
    """The adapter of every request; every fifth of a larger batch has none."""
    return [-1 if i % 5 == 4 else i % case["adapters"] for i in range(case["requests"])]


def work(case):
    new = _new(case)
    T, R = sum(new), len(new)
    if case["op"] == "plan":
        # lengths, counts and parents in; starts, slots, positions, masks and new table entries out
        return dict(bytes=12 * R + T * (4 + 4 + (12 if case["tree"] else 0)) + 8 * (T // case["page"] + R), flops=0)
    if case["op"] == "append":
        row = (case["heads"] + 2 * case["kv"]) * case["dim"] * 2
        return dict(bytes=T * (2 * row + 8 + 2 * case["dim"]), flops=T * (case["heads"] + case["kv"]) * case["dim"] * 3)
    if case["op"] == "attend":
        kv, h, d, lens = case["kv"], case["heads"], case["dim"], _lens(case)
        keys = sum(l + n for l, n in zip(lens, new))
        # a row's own tree counts as half of it: a chain's rows see that much
        seen = sum(n * (l + (n + 1) // 2) for l, n in zip(lens, new))
        return dict(bytes=keys * kv * d * 4 + T * h * d * 4 + 4 * (keys // case["page"]), flops=4 * seen * h * d)
    if case["op"] == "keep":
        moved = sum(min(max(n - 1, 0), case["kept"]) for n in new)
        return dict(bytes=moved * case["layers"] * 2 * case["kv"] * case["dim"] * 4 + 16 * R, flops=0)
    of, ranks = _adapter_of(case), _ranks(case)
    used = sum(ranks[a] for a in set(of) if a >= 0)
    seen = sum(n * ranks[a] for n, a in zip(new, of) if a >= 0)
    K, N = case["K"], case["N"]
    return dict(bytes=T * K * 2 + used * (K + N) * 2 + T * N * (2 + (4 if case["base"] == "f32" else 2)) + 4 * T, flops=2 * seen * (K + N))


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(lens, page, gen, spare=0, width=0):
    """A block table for requests of `lens` tokens, its pages in a random order, and the pages that it leaves free."""
    held = [-(-l // page) for l in lens]
    width, n = width or max(held) + spare, sum(held)
    pages = torch.randperm(n + spare * len(lens), device="cuda", generator=gen).to(torch.int32)
    col = torch.arange(width, device="cuda")[None]
    start = torch.tensor([0] + held[:-1], device="cuda").cumsum(0)[:, None]
    mine = col < torch.tensor(held, device="cuda")[:, None]
    table = torch.where(mine, pages[(start + col).clamp(max=pages.numel() - 1)], -1).to(torch.int32)
    return table, pages[n:].contiguous()


def _parents(new, gen):
    """Random trees: the parent of drafted token j is one of the seven before it, or the last cached token (-1)."""
    j = torch.cat([torch.arange(n, device="cuda") for n in new]) if sum(new) else torch.zeros(0, device="cuda")
    back = (torch.rand(j.numel(), device="cuda", generator=gen) * 7).floor() + 1
    return (j - back).clamp(min=-1).to(torch.int32)


def _reach(parents, q_start, n_max):
    """[R, n_max, n_max]: whether drafted token i of a request comes from token j or is it (the closure of its parents)."""
    new = (q_start[1:] - q_start[:-1]).long()
    j = torch.arange(n_max, device=parents.device)
    mine = j[None] < new[:, None]
    p = parents.long()[(q_start[:-1, None].long() + j[None]).clamp(max=max(parents.numel() - 1, 0))]
    step = ((p[:, :, None] == j) & mine[:, :, None]).float()
    return (torch.linalg.matrix_power(step + torch.eye(n_max, device=parents.device), max(n_max, 1)) > 0) & mine[:, :, None], mine


def _bits(reach):
    return (reach.long() << torch.arange(reach.shape[-1], device=reach.device)).sum(-1)


def prepare(case, seed):
    gen = _gen(seed)
    new = _new(case)
    R, T = len(new), sum(new)
    s = dict(case=case, T=T, n_max=max(new), q_start=_i32([sum(new[:i]) for i in range(R + 1)]))
    dt = DTYPES[case.get("dtype", "bf16")]

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dt)

    if case["op"] == "plan":
        rng = random.Random(seed)
        lens = [rng.randint(0, case["len_hi"]) for _ in range(R)]
        more = -(-case["new_hi"] // case["page"]) + 1
        table, free = _table([max(l, 1) for l in lens], case["page"], gen, more, width=-(-case["len_hi"] // case["page"]) + more)
        s.update(lens=_i32(lens), new=_i32(new), table=table, free=free, count=_i32([free.numel()]), count_out=_i32([0]),
                 parents=_parents(new, gen) if case["tree"] else None)
        return s
    if case["op"] == "lora":
        n, r, K, N = case["adapters"], case["rank_max"], case["K"], case["N"]
        base = torch.randn((T, N), device="cuda", generator=gen)
        s.update(x=randn(T, K), A=randn(n, r, K, scale=K ** -0.5), B=randn(n, N, r, scale=0.1),
                 scales=torch.rand(n, device="cuda", generator=gen) + 0.5, ranks=_i32(_ranks(case)),
                 idx=torch.repeat_interleave(_i32(_adapter_of(case)), torch.tensor(new, device="cuda")),
                 base=base if case["base"] == "f32" else base.to(dt), out=torch.zeros((T, N), dtype=dt, device="cuda"))
        return s
    lens = _lens(case)
    kv, dim, page = case["kv"], case["dim"], case["page"]
    table, free = _table([l + n for l, n in zip(lens, new)], page, gen, spare=1 if case["op"] == "keep" else 0)
    pages = int(table.max()) + 1 if case["op"] != "keep" else int((table >= 0).sum()) + free.numel()
    s.update(lens=_i32(lens), table=table, pages=pages, len_max=max(l + n for l, n in zip(lens, new)))
    if case["op"] == "keep":
        # the accepted path of every request: up to `kept` drafted tokens that follow one another, the first one dropped
        kept = [min(max(n - 1, 0), case["kept"]) for n in new]
        rng = random.Random(seed)
        path = [sorted(rng.sample(range(1, n), k)) + [0] * (n - k) if k else [0] * n for n, k in zip(new, kept)]
        space = torch.zeros(pages, dtype=torch.int32, device="cuda")
        space[:free.numel()] = free
        s.update(kv=randn(case["layers"], 2, pages, page, kv, dim), kept=_i32(kept), path=_i32([p for q in path for p in q]), free=space,
                 count=_i32([free.numel()]), lens_out=_i32([0] * R), count_out=_i32([0]))
        return s
    heads = case["heads"]
    if case["op"] == "append":
        j = torch.cat([torch.arange(n, device="cuda") for n in new])
        req = torch.repeat_interleave(torch.arange(R, device="cuda"), torch.tensor(new, device="cuda"))
        pos = s["lens"][req] + j
        slots = table[req, pos // page].long() * page + pos % page
        # rows of a fused projection: Q, K and V are column slices; angles as in a table of [cos | sin] rows
        angle = torch.arange(s["len_max"], device="cuda", dtype=torch.float64)[:, None] * 500000.0 ** (
            -torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
        qkv = randn(T, (heads + 2 * kv) * dim)
        q, k, v = qkv.split([heads * dim, kv * dim, kv * dim], 1)
        s.update(q=q.unflatten(1, (heads, dim)), k=k.unflatten(1, (kv, dim)), v=v.unflatten(1, (kv, dim)),
                 lut=torch.cat([angle.cos(), angle.sin()], 1).to(torch.bfloat16), positions=pos.to(torch.int32),
                 slots=slots.to(torch.int32), cache=randn(2, pages, page, kv, dim), q_out=torch.zeros((T, heads, dim), dtype=dt, device="cuda"))
        return s
    mask = None
    if case["tree"]:
        reach, mine = _reach(_parents(new, gen), s["q_start"], s["n_max"])
        mask = _bits(reach)[mine]
    s.update(q=randn(T, heads, dim, scale=1.5), cache=randn(2, pages, page, kv, dim), mask=mask, scale=dim ** -0.5,
             out=torch.zeros((T, heads, dim), dtype=dt, device="cuda"))
    return s


# ---- the plain forms -------------------------------------------------------------------------------
def _plain_plan(s):
    c, lens, new, table, T = s["case"], s["lens"].long(), s["new"].long(), s["table"], s["T"]
    page, dev = c["page"], lens.device
    held = (lens + page - 1) // page
    need = (lens + new + page - 1) // page - held
    # the i-th new page of a request comes from the top of the free pages, the requests one after another
    first = need.cumsum(0) - need
    i = torch.arange(table.shape[1], device=dev)[None] - held[:, None]
    taken = s["free"][(s["count"].long() - 1 - first[:, None] - i).clamp(0, s["free"].numel() - 1)]
    table.copy_(torch.where((i >= 0) & (i < need[:, None]), taken, table))
    end = new.cumsum(0)
    q_start = torch.cat([end.new_zeros(1), end])
    t = torch.arange(T, device=dev)
    req = torch.searchsorted(end, t, right=True)
    j = t - q_start[req]
    at = lens[req] + j
    slots = table[req, at // page].long() * page + at % page
    positions, mask = at, None
    if c["tree"]:
        reach, mine = _reach(s["parents"], q_start, max(s["n_max"], 1))
        mask = _bits(reach)[mine]
        positions = lens[req] + (reach.sum(-1) - 1)[mine]
    s["count_out"].copy_(s["count"] - need.sum())
    out = [q_start.int(), slots.int(), positions.int(), table, s["count_out"]]
    return out + [mask] if c["tree"] else out


def _rotate(x, lut):
    """[T, heads, dim] by a [cos | sin] row of each token, halves against each other."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    cos, sin = lut[:, None, :half], lut[:, None, half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_append(s):
    lut, dt = s["lut"][s["positions"].long()].float(), s["q"].dtype
    flat = s["cache"].flatten(1, 2)
    at = s["slots"].long()
    s["q_out"].copy_(_rotate(s["q"].float(), lut).to(dt))
    flat[0, at] = _rotate(s["k"].float(), lut).to(dt)
    flat[1, at] = s["v"]
    return s["q_out"], s["cache"]


def _plain_attend(s):
    c, q_start, lens = s["case"], s["q_start"].long(), s["lens"].long()
    page, kv, dim, L, n = c["page"], c["kv"], c["dim"], s["len_max"], s["n_max"]
    dev, group = lens.device, c["heads"] // c["kv"]
    new = q_start[1:] - q_start[:-1]
    # every request padded to the longest: keys [R, L, kv, dim], queries [R, n, kv, group, dim]
    p = torch.arange(L, device=dev)
    page_of = s["table"][:, p // page].long().clamp(min=0) * page + p % page
    k, v = (x.flatten(0, 1)[page_of].float() for x in s["cache"])
    j = torch.arange(n, device=dev)
    mine = j[None] < new[:, None]
    row = torch.where(mine, q_start[:-1, None] + j, 0)
    q = s["q"][row].float().view(-1, n, kv, group, dim) * s["scale"]
    score = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(-1, kv, n * group, dim), k.permute(0, 2, 3, 1)).view(-1, kv, n, group, L)
    drafted = p[None] - lens[:, None]
    if s["mask"] is None:
        seen = drafted[:, None, :] <= j[None, :, None]
    else:
        bit = (s["mask"][row][:, :, None] >> drafted[:, None, :].clamp(0, 63)) & 1
        seen = (drafted[:, None, :] < 0) | ((drafted[:, None, :] < new[:, None, None]) & (bit == 1))
    seen = seen[:, None, :, None, :]
    top = torch.where(seen, score, -math.inf).amax(-1, keepdim=True)
    weight = torch.where(seen, torch.exp(score - torch.where(top > -math.inf, top, 0.0)), 0.0)
    total = weight.sum(-1, keepdim=True)
    weight = weight / torch.where(total > 0, total, 1.0)
    o = torch.matmul(weight.view(-1, kv, n * group, L), v.permute(0, 2, 1, 3)).view(-1, kv, n, group, dim)
    s["out"][row[mine]] = o.permute(0, 2, 1, 3, 4).reshape(-1, n, kv * group, dim)[mine].to(s["out"].dtype)
    return s["out"]


def _plain_keep(s):
    page, table, q_start, lens, kept = s["case"]["page"], s["table"], s["q_start"].long(), s["lens"].long(), s["kept"].long()
    new = q_start[1:] - q_start[:-1]
    req = torch.repeat_interleave(torch.arange(lens.numel(), device=lens.device), kept, output_size=None)
    i = torch.arange(req.numel(), device=lens.device) - (kept.cumsum(0) - kept)[req]
    src, dst = lens[req] + s["path"].long()[q_start[req] + i], lens[req] + i
    flat = s["kv"].flatten(2, 3)
    flat[:, :, table[req, dst // page].long() * page + dst % page] = flat[:, :, table[req, src // page].long() * page + src % page]
    after = lens + kept
    had, has = (lens + new + page - 1) // page, (after + page - 1) // page
    gone = had - has
    r2 = torch.repeat_interleave(torch.arange(lens.numel(), device=lens.device), gone)
    k = torch.arange(r2.numel(), device=lens.device)
    s["free"][s["count"].long() + k] = table[r2, has[r2] + k - (gone.cumsum(0) - gone)[r2]]
    s["lens_out"].copy_(after)
    s["count_out"].copy_(s["count"] + gone.sum())
    return s["kv"], s["lens_out"], s["free"], s["count_out"]


def _plain_lora(s):
    n, r, K = s["A"].shape
    T, of = s["T"], s["idx"].long()
    # through every adapter, then each row's own part of it
    low = torch.matmul(s["x"].float(), s["A"].float().view(n * r, K).t()).view(T, n, r)
    own_part = (torch.arange(n, device=of.device) == of[:, None])[:, :, None] & (torch.arange(r, device=of.device) < s["ranks"][:, None])
    low = torch.where(own_part, low * s["scales"][:, None], 0.0).view(T, n * r)
    up = torch.matmul(low, s["B"].float().permute(0, 2, 1).reshape(n * r, -1))
    s["out"].copy_((s["base"].float() + up).to(s["out"].dtype))
    return s["out"]


_PLAIN = dict(plan=_plain_plan, append=_plain_append, attend=_plain_attend, keep=_plain_keep, lora=_plain_lora)


# ---- the framework's calls ---------------------------------------------------------------------------
def _run_own(s):
    from mlir_air_b200 import ops
    c = s["case"]
    if "ws" not in s:  # what a program makes once, at its start
        s["ws"] = ops.RequestWorkspace()
        if c["op"] == "lora":
            s["adapters"] = ops.LoraAdapters(s["A"], s["B"], s["scales"], s["ranks"])
        if c["op"] in ("append", "attend"):
            s["layer"] = ops.KVCache(*s["cache"])
    if c["op"] == "plan":
        p = ops.page_plan(s["lens"], s["new"], s["table"], s["free"], s["count"], c["page"], s["T"], s["ws"], parents=s["parents"],
                          free_count_out=s["count_out"])
        out = [p.q_start, p.slots, p.positions, s["table"], s["count_out"]]
        return out + [p.mask] if c["tree"] else out
    if c["op"] == "append":
        ops.rope_append(s["q"], s["k"], s["v"], s["lut"], s["positions"], s["slots"], s["layer"], s["ws"], q_out=s["q_out"])
        return s["q_out"], s["cache"]
    if c["op"] == "attend":
        return ops.tree_attention(s["q"], s["layer"], s["table"], s["lens"], s["q_start"], s["ws"], mask=s["mask"], scale=s["scale"],
                                  out=s["out"])
    if c["op"] == "keep":
        ops.page_keep(s["kv"], s["table"], s["lens"], s["q_start"], s["kept"], s["free"], s["count"], s["ws"], path=s["path"],
                      lens_out=s["lens_out"], free_count_out=s["count_out"])
        return s["kv"], s["lens_out"], s["free"], s["count_out"]
    return ops.lora(s["x"], s["adapters"], s["idx"], s["base"], s["ws"], out=s["out"])


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- 64 bits, from the definitions, request by request ---------------------------------------------------
def exact(case, seed):
    if case["op"] == "plan":  # whole numbers
        return None
    s = prepare(case, seed)
    new, starts = _new(case), s["q_start"].tolist()
    if case["op"] == "lora":
        out = s["base"].double()
        for i, a in enumerate(_adapter_of(case)):
            if a >= 0:
                rows, r = slice(starts[i], starts[i + 1]), int(s["ranks"][a])
                out[rows] += float(s["scales"][a]) * (s["x"][rows].double() @ s["A"][a, :r].double().T) @ s["B"][a, :, :r].double().T
        return out
    lens, page = s["lens"].tolist(), case["page"]

    def slots(r, first, last):
        at = torch.arange(first, last, device="cuda")
        return s["table"][r].long()[at // page] * page + at % page

    if case["op"] == "keep":
        kv, where = s["kv"].double(), s["path"].tolist()
        rows = kv.flatten(2, 3)
        for r, k in enumerate(s["kept"].tolist()):
            mine = rows[:, :, slots(r, lens[r], lens[r] + new[r])]
            for i in range(k):
                rows[:, :, slots(r, lens[r] + i, lens[r] + i + 1)] = mine[:, :, where[starts[r] + i], None]
        return kv, None, None, None
    if case["op"] == "append":
        q, cache, half = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), s["cache"].double(), case["dim"] // 2
        for r in range(len(new)):
            rows, at = slice(starts[r], starts[r + 1]), slots(r, lens[r], lens[r] + new[r])
            turn = s["lut"][lens[r]:lens[r] + new[r]].double()
            turn = torch.complex(turn[:, :half], turn[:, half:])[:, None]
            for src, dst, where in ((s["q"], q, rows), (s["k"], cache[0].flatten(0, 1), at)):
                z = torch.complex(src[rows, :, :half].double(), src[rows, :, half:].double()) * turn
                dst[where] = torch.cat([z.real, z.imag], -1)
            cache[1].flatten(0, 1)[at] = s["v"][rows].double()
        return q, cache
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for r in range(len(new)):
        at = slots(r, 0, lens[r] + new[r])
        k, v = (x.flatten(0, 1)[at].double() for x in s["cache"])
        hidden = torch.zeros((new[r], lens[r] + new[r]), dtype=torch.bool, device="cuda")
        own_tree = torch.ones((new[r], new[r]), dtype=torch.bool, device="cuda").tril()
        if s["mask"] is not None:
            own_tree = (s["mask"][starts[r]:starts[r + 1], None] >> torch.arange(new[r], device="cuda")) % 2 != 0
        hidden[:, lens[r]:] = ~own_tree
        group = case["heads"] // case["kv"]
        for h in range(case["heads"]):
            score = s["q"][starts[r]:starts[r + 1], h].double() @ k[:, h // group].T * s["scale"]
            out[starts[r]:starts[r + 1], h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1).nan_to_num(0.0) @ v[:, h // group]
    return out
