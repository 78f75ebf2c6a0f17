"""tree_attention against 64 bits: head layouts, page and tile borders, masks, strides, values that no row sees."""
import math

import pytest
import torch

from request_util import attend_ref, i32, make_table, random_masks, starts

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def run(lens, new, H, kv, D, page, dtype=BF, tree=False, empty=0.0, seed=0, scale=None, q_scale=1.5):
    from mlir_air_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    T = sum(new)
    table, pages = make_table([l + n for l, n in zip(lens, new)], page, seed, extra=2)
    k, v = (rnd(pages, page, kv, D).to(dtype) for _ in range(2))
    q = (rnd(T, H, D) * q_scale).to(dtype)
    mask = random_masks(new, seed, empty) if tree else None
    # slots that no request's token lies in hold NaN
    used = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
    for r, (l, n) in enumerate(zip(lens, new)):
        p = torch.arange(l + n, device="cuda")
        used[table[r, p // page].long(), p % page] = True
    k[~used] = float("nan")
    v[~used] = float("nan")
    ws = ops.RequestWorkspace()
    sc = D ** -0.5 if scale is None else scale
    out = ops.tree_attention(q, ops.KVCache(k, v), table, i32(lens), i32(starts(new)), ws, mask=mask, scale=scale)
    ws.check()
    ref, tol = attend_ref(q, k.nan_to_num(), v.nan_to_num(), table, lens, new, mask, sc)
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()} values are off, at most {float((err / tol.clamp(min=1e-30)).max()):.2f} times"
    return out


@pytest.mark.parametrize("H,kv", [(1, 1), (8, 8), (8, 2), (8, 1), (10, 2), (12, 12), (16, 2), (36, 12)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_layouts(H, kv, D):
    run([37, 0, 130], [1, 3, 2], H, kv, D, 16)


@pytest.mark.parametrize("D", [16, 48, 80, 96, 160, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_other_head_sizes(D, dtype):
    run([37, 0, 70], [1, 3, 6], 4, 2, D, 16, dtype, tree=True)


@pytest.mark.parametrize("D", [16, 32, 96, 112, 144, 208, 256])
@pytest.mark.parametrize("lens,new", [([5000], [1]), ([700, 0, 33, 129], [1, 64, 0, 17]), ([0, 3], [70, 1])])
def test_other_head_sizes_over_long_contexts(D, lens, new):
    run(lens, new, 8, 2, D, 16, FP if D % 32 else BF, tree=max(new) <= 64, empty=0.1)


@pytest.mark.parametrize("D,wide", [(48, 64), (96, 104), (112, 128), (160, 168)])
def test_columns_behind_a_head_are_left(D, wide):
    """Heads that are slices of wider rows: what lies behind them is not used (NaN) and not written (7)."""
    from mlir_air_b200 import ops
    lens, new, H, kv, page = [70, 5, 0], [3, 20, 1], 4, 2, 8
    gen = torch.Generator(device="cuda").manual_seed(3)
    table, pages = make_table([l + n for l, n in zip(lens, new)], page, 3)
    wide_of = lambda *s: torch.full((*s, wide), float("nan"), device="cuda", dtype=BF)  # noqa: E731
    k, v, q = wide_of(pages, page, kv)[..., :D], wide_of(pages, page, kv)[..., :D], wide_of(sum(new), H)[..., :D]
    for x in (k, v, q):
        x.copy_(torch.randn(x.shape, device="cuda", generator=gen))
    mask, ws = random_masks(new, 3), ops.RequestWorkspace()
    k[table[1, 1], 0, 0, 3], v[table[1, 1], 2, 1, 5] = 3.0, float("inf")  # (a drafted token that some rows see: infinite for them only)
    into = torch.full((sum(new), H, wide), 7.0, device="cuda", dtype=BF)
    ops.tree_attention(q, ops.KVCache(k, v), table, i32(lens), i32(starts(new)), ws, mask=mask, out=into[..., :D])
    ws.check()
    assert bool((into[..., D:] == 7).all())
    out = into[..., :D]
    j = (int(table[1, 1]), 8 + 2 - lens[1])  # its page, and its place among the request's new tokens
    sees = ((mask[3:23] >> j[1]) & 1).bool()
    rows = torch.arange(3, 23, device="cuda")
    assert bool(torch.isinf(out[rows[sees]][:, 2:, 5]).all()) and 0 < int(sees.sum()) < 20
    out[rows[sees], 2:, 5] = 0
    v[j[0], 2, 1, 5] = 0
    ref, tol = attend_ref(q, k, v, table, lens, new, mask, D ** -0.5)
    ref[rows[sees], 2:, 5] = 0
    assert bool(((out.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("page", [1, 3, 8, 16, 64, 128, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_pages(page, D):
    run([0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200], [1, 2, 1, 1, 3, 1, 1, 64, 5, 1, 2, 0], 4, 2, D, page, tree=True)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("new", [[1], [2], [16], [17], [33], [64], [64, 1, 30, 0, 7]])
@pytest.mark.parametrize("H,kv,D", [(8, 1, 128), (4, 4, 64), (6, 2, 128)])
def test_trees(dtype, new, H, kv, D):
    run([300 + 11 * i for i in range(len(new))], new, H, kv, D, 16, dtype, tree=True)


@pytest.mark.parametrize("H,kv,D", [(8, 2, 128), (4, 1, 64)])
@pytest.mark.parametrize("lens,new", [([0], [1]), ([0], [130]), ([100, 0, 7], [200, 65, 129]), ([1], [300])])
def test_chains_longer_than_a_tree(H, kv, D, lens, new):
    run(lens, new, H, kv, D, 16)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_see_nothing(D):
    out = run([0, 50, 0], [9, 20, 1], 4, 2, D, 16, tree=True, empty=0.5)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("D,H,kv", [(64, 8, 2), (128, 8, 1), (128, 32, 4)])
@pytest.mark.parametrize("lens,new", [([5000], [1]), ([3001, 12], [4, 1]), ([2500, 2500], [33, 64]), ([9000], [20])])
def test_long_contexts_are_split_and_joined(D, H, kv, lens, new):
    run(lens, new, H, kv, D, 64, tree=True)


def test_many_requests_of_all_lengths():
    lens = [(i * 37) % 500 for i in range(150)]
    run(lens, [(i * 7) % 5 for i in range(150)], 8, 2, 128, 16, tree=True)


@pytest.mark.parametrize("H,kv", [(2, 1), (24, 1)])
@pytest.mark.parametrize("n", [128, 129, 300, 1000, 4096])
def test_as_many_requests_as_there_may_be(n, H, kv):
    run([(i * 37) % 90 for i in range(n)], [0 if i % 50 < 40 and i > n // 2 else 1 + (i % 9 == 0) for i in range(n)], H, kv, 64, 16)


@pytest.mark.parametrize("q_scale", [0.0, 12.0, 60.0])
def test_flat_and_peaked_scores(q_scale):
    run([700, 40], [5, 1], 8, 2, 128, 16, tree=True, q_scale=q_scale)


def test_a_negative_scale():
    run([100], [3], 4, 2, 64, 16, scale=-0.3)


def _small(seed=0, D=128, new=(3, 20), lens=(40, 75), page=16, H=8, kv=2):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    table, pages = make_table([l + n for l, n in zip(lens, new)], page, seed)
    k, v = (torch.randn((pages, page, kv, D), device="cuda", generator=gen).to(BF) for _ in range(2))
    q = torch.randn((sum(new), H, D), device="cuda", generator=gen).to(BF)
    return q, k, v, table, i32(lens), i32(starts(new)), random_masks(new, seed)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,lens", [((3, 20), (40, 75)), ((1, 1), (40, 300)), ((64, 64), (400, 3))])
def test_strides_do_not_matter(D, new, lens):
    from mlir_air_b200 import ops
    q, k, v, table, ln, st, mask = _small(D=D, new=new, lens=lens)
    T, H = q.shape[:2]
    ws = ops.RequestWorkspace()
    want = ops.tree_attention(q, ops.KVCache(k, v), table, ln, st, ws, mask=mask)
    # q a column slice of a projection, out a slice of a wider buffer, heads in front of slots, K and V in one tensor, a table in a wider one
    wide = torch.full((T, H * D + 64), float("nan"), device="cuda").to(BF)
    wide[:, 32:32 + H * D] = q.flatten(1)
    both = torch.stack([k.transpose(1, 2), v.transpose(1, 2)], 1).contiguous()
    t2 = torch.full((table.shape[0], table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    t2[:, :table.shape[1]] = table
    out = torch.full((T, H + 3, D + 8), 7.0, device="cuda").to(BF)
    got = ops.tree_attention(wide[:, 32:32 + H * D].unflatten(1, (H, D)), ops.KVCache(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)),
                             t2[:, :table.shape[1]], ln, st, ws, mask=mask, out=out[:, 1:1 + H, :D])
    ws.check()
    assert torch.equal(got, want)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 1 + H:] == 7).all()) and bool((out[..., D:] == 7).all())


@pytest.mark.parametrize("new,lens", [((3, 20), (40, 75)), ((1, 1), (40, 300)), ((64, 64), (400, 3))])
def test_values_no_row_sees_do_not_matter(new, lens):
    """Infinities and NaN in a drafted token that a row's mask leaves out change nothing for that row."""
    from mlir_air_b200 import ops
    q, k, v, table, ln, st, _ = _small(new=new, lens=lens)
    ws = ops.RequestWorkspace()
    s = starts(list(new))
    mask = torch.zeros(sum(new), dtype=torch.int64, device="cuda")
    for r, n in enumerate(new):
        for j in range(n):
            mask[s[r] + j] = 1 << j if j < 63 else -2 ** 63
    mask[s[1] - 1] = 0  # the last token of the first request is seen by no one
    want = ops.tree_attention(q, ops.KVCache(k, v), table, ln, st, ws, mask=mask)
    for bad in (float("nan"), float("inf"), -float("inf")):
        k2, v2 = k.clone(), v.clone()
        p = lens[0] + new[0] - 1
        k2[int(table[0, p // 16]), p % 16] = bad
        v2[int(table[0, p // 16]), p % 16] = bad
        assert torch.equal(ops.tree_attention(q, ops.KVCache(k2, v2), table, ln, st, ws, mask=mask), want)
        # seen by one row: that row is not finite, the others are as before
        if new[0] > 1:
            m2 = mask.clone()
            m2[s[0]] |= 1 << (new[0] - 1) if new[0] < 64 else -2 ** 63
            got = ops.tree_attention(q, ops.KVCache(k, v2), table, ln, st, ws, mask=m2)
            ref = ops.tree_attention(q, ops.KVCache(k, v), table, ln, st, ws, mask=m2)
            assert not torch.isfinite(got[s[0]]).any()
            assert torch.equal(got[s[0] + 1:], ref[s[0] + 1:])
    ws.check()


def test_rows_behind_the_last_request_are_left():
    from mlir_air_b200 import ops
    q, k, v, table, ln, st, mask = _small()
    ws = ops.RequestWorkspace()
    T = q.shape[0]
    pad = lambda t: torch.cat([t, torch.full_like(t[:5], float("nan") if t.is_floating_point() else -1)])  # noqa: E731
    out = torch.full((T + 5, 8, 128), 3.0, device="cuda").to(BF)
    ops.tree_attention(pad(q), ops.KVCache(k, v), table, ln, st, ws, mask=pad(mask), out=out)
    assert torch.equal(out[:T], ops.tree_attention(q, ops.KVCache(k, v), table, ln, st, ws, mask=mask)) and bool((out[T:] == 3).all())
    fresh = ops.tree_attention(pad(q), ops.KVCache(k, v), table, ln, st, ws, mask=pad(mask))
    assert bool((fresh[T:] == 0).all())
    ws.check()


@pytest.mark.parametrize("D,new,lens", [(64, (1, 3), (2000, 9)), (128, (40, 64), (900, 30)), (96, (5, 1), (700, 3)), (160, (4, 1), (300, 3))])
def test_the_rows_may_be_overwritten(D, new, lens):
    from mlir_air_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(5)
    table, pages = make_table([l + n for l, n in zip(lens, new)], 16, 5)
    k, v = (torch.randn((pages, 16, 2, D), device="cuda", generator=gen).to(BF) for _ in range(2))
    q = torch.randn((sum(new), 8, D), device="cuda", generator=gen).to(BF)
    args, ws = (ops.KVCache(k, v), table, i32(lens), i32(starts(new))), ops.RequestWorkspace()
    want = ops.tree_attention(q, *args, ws)
    assert ops.tree_attention(q, *args, ws, out=q) is q and torch.equal(q, want)
    ws.check()


def test_the_same_bits_every_time():
    from mlir_air_b200 import ops
    for new, lens in (((1,) * 5, (3000, 10, 700, 64, 9000)), ((64, 20), (5000, 800))):
        q, k, v, table, ln, st, mask = _small(new=new, lens=lens)
        ws = ops.RequestWorkspace()
        first = ops.tree_attention(q, ops.KVCache(k, v), table, ln, st, ws, mask=mask)
        for _ in range(5):
            assert torch.equal(ops.tree_attention(q, ops.KVCache(k, v), table, ln, st, ws, mask=mask), first)


def test_slots_beyond_32_bit_offsets():
    """A cache of more than 2^31 elements: the last pages are reached, not the wrapped ones."""
    from mlir_air_b200 import ops
    page, kv, D = 128, 8, 128
    pages = 2 ** 31 // (page * kv * D) + 3
    k = torch.zeros((pages, page, kv, D), dtype=BF, device="cuda")
    v = torch.zeros_like(k)
    gen = torch.Generator(device="cuda").manual_seed(1)
    for c in (k, v):
        c[-2:] = torch.randn((2, page, kv, D), device="cuda", generator=gen).to(BF)
    ws = ops.RequestWorkspace()
    for n in (1, 40):
        q = torch.randn((n, 16, D), device="cuda", generator=gen).to(BF)
        args = (i32([200]), i32([0, n]), ws)
        far = ops.tree_attention(q, ops.KVCache(k, v), i32([[pages - 1, pages - 2]]), *args)
        near = ops.tree_attention(q, ops.KVCache(k[-2:].clone(), v[-2:].clone()), i32([[1, 0]]), *args)
        assert torch.equal(far, near) and bool(far.abs().sum() > 0)
    ws.check()


def test_bad_pages_lengths_and_starts_are_reported():
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    for new, lens in (((3, 20), (40, 75)), ((1, 1), (40, 300)), ((64, 64), (400, 3))):
        q, k, v, table, ln, st, mask = _small(new=new, lens=lens)
        ws = ops.RequestWorkspace()
        cache = ops.KVCache(k, v)
        good = ops.tree_attention(q, cache, table, ln, st, ws, mask=mask)
        ws.check()
        for page in (-1, k.shape[0], 2 ** 31 - 1):
            t2 = table.clone()
            t2[0, 1] = page
            got = ops.tree_attention(q, cache, t2, ln, st, ws, mask=mask)
            assert torch.equal(got[new[0]:], good[new[0]:])  # the other request is not touched
            with pytest.raises(AwqBackendError, match="page outside the cache"):
                ws.check()
            ws.check()  # reported once
        for l2, s2 in ((i32([-1, lens[1]]), st), (i32([2 ** 31 - 1, lens[1]]), st), (ln, i32([0, q.shape[0] + 1, q.shape[0]])), (ln, i32([-5, 2, 3]))):
            ops.tree_attention(q, cache, table, l2, s2, ws, mask=mask)
            with pytest.raises(AwqBackendError, match="tree_attention: lengths or starts"):
                ws.check()
        assert torch.equal(ops.tree_attention(q, cache, table, ln, st, ws, mask=mask), good)
        ws.check()


def test_streams_graphs_and_no_rows():
    from mlir_air_b200 import ops
    q, k, v, table, ln, st, mask = _small(new=(3, 20), lens=(4000, 75))
    cache, ws = ops.KVCache(k, v), ops.RequestWorkspace()
    want = ops.tree_attention(q, cache, table, ln, st, ws, mask=mask)
    torch.cuda.synchronize()
    side, ws2 = torch.cuda.Stream(), ops.RequestWorkspace()
    out = torch.zeros_like(want)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.tree_attention(q, cache, table, ln, st, ws2, mask=mask, out=out)
    again = ops.tree_attention(q, cache, table, ln, st, ws, mask=mask)  # at the same time, on a workspace of its own
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tree_attention(q, cache, table, ln, st, ws, mask=mask, out=out)
    q2 = torch.randn_like(q)
    want2 = ops.tree_attention(q2, cache, table, i32([100, 9]), st, ws, mask=mask)
    q.copy_(q2)
    ln.copy_(i32([100, 9]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want2)
    empty = ops.tree_attention(q[:0], cache, table[:0], ln[:0], st[:1], ws)
    assert empty.shape == (0, 8, 128)
    ws.check()
    ws2.check()


def test_arguments_that_do_not_fit_are_refused():
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    q, k, v, table, ln, st, mask = _small()
    cache, ws = ops.KVCache(k, v), ops.RequestWorkspace()
    ok = dict(q=q, cache=cache, table=table, lens=ln, q_start=st, ws=ws, mask=mask)
    wrong = [dict(q=q[:, :7]), dict(q=q.half()), dict(q=q[..., :64]), dict(q=q.cpu()), dict(q=q[0]), dict(table=table.long()), dict(table=table[:1]),
             dict(lens=ln.long()), dict(lens=ln[:1]), dict(q_start=st[:2]), dict(mask=mask[:-1]), dict(mask=mask.int()), dict(out=q.float()),
             dict(out=q[:-1]), dict(scale=float("nan")), dict(scale=float("inf"))]
    for change in wrong:
        with pytest.raises(AwqBackendError):
            ops.tree_attention(**{**ok, **change})
    odd = torch.zeros(q.numel() + 1, dtype=BF, device="cuda")[1:].view_as(q)
    with pytest.raises(AwqBackendError, match="16-byte"):
        ops.tree_attention(**{**ok, "q": odd})
    with pytest.raises(AwqBackendError, match="multiples of 8"):
        ops.tree_attention(**{**ok, "q": torch.zeros((q.shape[0], 8, 132), dtype=BF, device="cuda")[..., :128]})
    for bad in ((k.float(), v.float()), (k, v.half()), (k, v[1:]), (k[..., :100], v[..., :100]), (k.cpu(), v.cpu()), (k[..., 0], v[..., 0]),
                (k[:0], v[:0]), (k.expand(-1, -1, 2, -1)[:, :1].expand(-1, 16, -1, -1), v)):
        with pytest.raises(AwqBackendError):
            ops.KVCache(*bad)
    ops.tree_attention(**ok)
    ws.check()


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("R,H,kv,D,n,length,page", [(64, 64, 8, 128, 60, 0, 16), (40, 32, 8, 64, 64, 0, 1), (150, 32, 8, 64, 20, 40, 16), (30, 24, 4, 64, 60, 70, 3)])
def test_values_that_are_not_finite_in_many_short_segments(R, H, kv, D, n, length, page, dtype, tree):
    """Infinities and NaN in new tokens of many requests, several segments of one tile or two to a CTA: a row that sees one has it in its result, all
    others are as near to 64 bits as without them."""
    from mlir_air_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(R)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    total = length + n
    table, pages = make_table([total] * R, page, R)
    k, v = (rnd(pages, page, kv, D).to(dtype) for _ in range(2))
    q = rnd(R * n, H, D).to(dtype)
    p = torch.arange(total, device="cuda")
    at = table[:, p // page].long(), (p % page)[None, :].expand(R, -1)
    mask = random_masks([n] * R, R) if tree else None
    new_seen = (mask.view(R, n, 1) >> torch.arange(n, device="cuda") & 1).bool() if tree else torch.ones((n, n), device="cuda").tril().bool().expand(R, n, n)
    seen = torch.cat([torch.ones((R, n, length), dtype=torch.bool, device="cuda"), new_seen], 2)
    # 64 bits, a cache head at a time
    ref, tol, u = [], [], torch.finfo(dtype).eps / 2
    for g in range(kv):
        kr, vr = k[at][:, :, g].double(), v[at][:, :, g].double()
        qr = q.view(R, n, kv, H // kv, D)[:, :, g].double()
        s = torch.einsum("rnhd,rpd->rhnp", qr, kr) * D ** -0.5
        w = torch.softmax(s.masked_fill(~seen[:, None], -torch.inf), -1)
        o, mag = torch.einsum("rhnp,rpd->rnhd", w, vr), torch.einsum("rhnp,rpd->rnhd", w, vr.abs())
        # (see attend_ref; the scores' part of the bound by the largest of all)
        d = D * 2.0 ** -24 * float(torch.einsum("rnhd,rpd->rhnp", qr.abs(), kr.abs()).max()) * D ** -0.5 + 2.0 ** -20
        ref.append(o)
        tol.append(u * o.abs() + (u + 2 * d) * mag + torch.finfo(dtype).smallest_normal * 2 * u)
    ref, tol = torch.stack(ref, 2), torch.stack(tol, 2) * 1.001  # [R, n, kv, H / kv, D]
    # one in three requests, some of its heads: a value of a token near the front, and of any
    extra = torch.zeros((R, n, kv, 1, D), dtype=torch.float64, device="cuda")
    host = torch.Generator().manual_seed(R)
    pick = lambda hi: int(torch.randint(0, hi, (1,), generator=host))  # noqa: E731
    planted = {}
    for r in range(0, R, 3):
        for what in (float("inf"), -float("inf"), float("nan"), float("inf")):
            j, g, e = (pick(4) if pick(2) else pick(n)), pick(kv), pick(D)
            v[at[0][r, length + j], at[1][r, length + j], g, e] = what
            planted[r, j, g, e] = what  # (a place drawn twice keeps the last)
    for (r, j, g, e), what in planted.items():
        extra[r, new_seen[r, :, j], g, 0, e] += what
    ws = ops.RequestWorkspace()
    args = (ops.KVCache(k, v), table, i32([length] * R), i32([n * r for r in range(R + 1)]), ws)
    for _ in range(3):
        out = ops.tree_attention(q, *args, mask=mask).view(R, n, kv, H // kv, D).double()
        ws.check()
        plain = (extra == 0).expand_as(out)
        assert bool(((out - ref).abs() <= tol)[plain].all())
        assert torch.equal(out[~plain].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0), extra.expand_as(out)[~plain].nan_to_num(nan=7.0, posinf=8.0, neginf=9.0))


@pytest.mark.parametrize("gap", [4.0, 14.0, 16.0, 17.5, 20.0])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,n,per_sm", [(64, 1, 3), (96, 1, 3), (128, 20, 2), (64, 20, 2), (160, 1, 1)])
def test_many_small_weights_behind_a_large_one(D, n, per_sm, dtype, gap):
    """Keys that hold all the weight and no value, and 32000 others `gap` nats below: what these add up to is the result.  As many requests over
    the same pages as CTAs run at once, so that a CTA, and each of its warps, has such a key and all of a request's others.

    With a = exp(-gap), m large keys and N others of value 1 the result is N a / (m + N a).  A weight is rounded by u, half a step, relative to
    itself, or in fp16, below 2^-21 of the largest, by half of 2^-31 of the largest: together N 2^-32 / m.  The rest as in attend_ref."""
    from mlir_air_b200 import ops
    R, group, page, length = (torch.cuda.get_device_properties(0).multi_processor_count * per_sm if D < 160 else 3), 4, 16, 32000
    k, v = torch.zeros((length // page + 2 * R, page, 1, D), dtype=dtype, device="cuda"), torch.ones((length // page + 2 * R, page, 1, D), dtype=dtype, device="cuda")
    for key in (0, 16, 32, 48):
        k[key // page, key % page, 0, 5], v[key // page, key % page] = gap, 0
    q = torch.zeros((R * n, group, D), dtype=dtype, device="cuda")
    q[..., 5] = 1
    blocks = length // page
    table = torch.arange(blocks + 2, dtype=torch.int32, device="cuda").repeat(R, 1)
    table[:, blocks:] = blocks + torch.arange(2 * R, dtype=torch.int32, device="cuda").view(R, 2)
    ws = ops.RequestWorkspace()
    out = ops.tree_attention(q, ops.KVCache(k, v), table, i32([length] * R), i32([n * r for r in range(R + 1)]), ws, scale=1.0)
    ws.check()
    a, m, u = math.exp(-gap), 4, torch.finfo(dtype).eps / 2
    others = length - m + 1 + torch.arange(n, dtype=torch.float64, device="cuda").repeat(R)
    want = (others * a / (m + others * a)).view(-1, 1, 1)
    d = D * 2.0 ** -24 * gap + 2.0 ** -20
    tol = u * want + (u + 2 * d) * want + (others.max() * 2.0 ** -32 / m if dtype == FP else 0) + torch.finfo(dtype).smallest_normal * 2 * u
    err = (out.double() - want).abs()
    assert bool((err <= tol * 1.001).all()), (float((err / want).max()), float((tol / want).max()))


@pytest.mark.parametrize("where", ["first keys", "last keys", "new token"])
@pytest.mark.parametrize("what", ["V nan", "V inf", "K nan"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,n", [(64, 1), (128, 1), (96, 1), (160, 1), (64, 33), (128, 33)])
def test_what_a_row_sees_reaches_it_whatever_its_weight(D, n, dtype, what, where):
    """NaN or infinity in a key that a row sees, but whose score lies so far below that its weight is 0 in 32 bits, alone or with all keys of its
    tile, its warp and its CTA: the result is not finite there (0 times infinity), and as it was elsewhere."""
    from mlir_air_b200 import ops
    length, page, group, kv, gap = 40000, 16, 2, 2, 200.0
    total = length + n
    gen = torch.Generator(device="cuda").manual_seed(D)
    table, pages = make_table([total], page, 1)
    k, v = torch.zeros((pages, page, kv, D), dtype=dtype, device="cuda"), torch.randn((pages, page, kv, D), device="cuda", generator=gen).to(dtype)
    at = lambda p: (int(table[0, p // page]), p % page)  # noqa: E731
    flat = table[0].long()[torch.arange(total, device="cuda") // page] * page + torch.arange(total, device="cuda") % page
    low = slice(0, length // 2) if where == "first keys" else slice(length // 2, length) if where == "last keys" else slice(length, length + 1)
    k.flatten(0, 1)[flat[low], :, 3] = -gap
    q = torch.zeros((n, kv * group, D), dtype=dtype, device="cuda")
    q[..., 3] = 1
    args = (table, i32([length]), i32([0, n]), ops.RequestWorkspace())
    was = ops.tree_attention(q, ops.KVCache(k, v), *args, scale=1.0)
    assert bool(torch.isfinite(was).all())
    page_at = at({"first keys": 777, "last keys": length - 333, "new token": length}[where])
    bad = torch.zeros(was.shape, dtype=torch.bool, device="cuda")
    if what == "K nan":
        k[page_at][1, 3] = float("nan")
        bad[:, group:] = True
    else:
        v[page_at][1, 17] = float(what[2:])
        bad[:, group:, 17] = True
    got = ops.tree_attention(q, ops.KVCache(k, v), *args, scale=1.0)
    args[-1].check()
    assert not bool(torch.isfinite(got[bad]).any()) and torch.equal(got[~bad], was[~bad])
