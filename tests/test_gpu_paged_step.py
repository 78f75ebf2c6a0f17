"""page_plan, rope_append and page_keep against plain forms; several steps of a serving loop in a row."""
import random

import pytest
import torch

from request_util import i32, make_table, starts

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def plan_ref(lens, new, table, free, count, page, T, parents=None):
    """The plan's definition, token by token, on host lists; table is changed in place."""
    st, slots, pos, mask = starts(new), [], [], []
    for r, (l, n) in enumerate(zip(lens, new)):
        held = -(-l // page)
        for b in range(held, -(-(l + n) // page)):
            count -= 1
            table[r][b] = free[count]
        for j in range(n):
            slots.append(table[r][(l + j) // page] * page + (l + j) % page)
            bits, depth, p = 1 << j, 0, j
            while parents is not None and parents[st[r] + p] >= 0:
                p = parents[st[r] + p]
                bits |= 1 << p
                depth += 1
            pos.append(l + (j if parents is None else depth))
            mask.append(bits - (1 << 64) if bits >> 63 else bits)
    pad = T - len(slots)
    return st, slots + [-1] * pad, pos + [0] * pad, mask + [0] * pad, count


def check_plan(lens, new, page, tree, seed=0, pad=0, spare=0):
    from mlir_air_b200 import ops
    rng = random.Random(seed)
    table, used = make_table([max(l, 0) for l in lens], page, seed, width=max(-(-(l + n) // page) for l, n in zip(lens, new)) + 1)
    need = sum(-(-(l + n) // page) - -(-l // page) for l, n in zip(lens, new))
    free = [used + i for i in range(need + spare)]
    rng.shuffle(free)
    pool = free + [-7] * used  # a stack of `pages` entries, the upper ones not in use
    T = sum(new) + pad
    parents = [rng.randint(max(-1, j - 4), j - 1) for n in new for j in range(n)] + [5] * pad if tree else None
    ws = ops.RequestWorkspace()
    count = i32([len(free)])
    host = table.tolist()
    want = plan_ref(lens, new, host, free, len(free), page, T, parents)
    lens_t = i32(lens)
    p = ops.page_plan(lens_t, i32(new), table, i32(pool), count, page, T, ws, parents=i32(parents) if tree else None)
    ws.check()
    assert p.q_start.tolist() == want[0] and p.slots.tolist() == want[1] and p.positions.tolist() == want[2]
    assert table.tolist() == host and count.tolist() == [want[4]] and lens_t.tolist() == list(lens)
    assert p.mask is None if not tree else p.mask.tolist() == want[3]


@pytest.mark.parametrize("page", [1, 5, 16, 128])
@pytest.mark.parametrize("tree", [False, True])
def test_plan(page, tree):
    check_plan([0, 1, 15, 16, 17, 300, 0, 31], [1, 0, 1, 1, 64, 33, 0, 2], page, tree, pad=7, spare=3)


@pytest.mark.parametrize("R,hi,tree", [(1, 1, False), (1, 64, True), (300, 8, True), (1000, 3, False), (4096, 2, True), (3, 20000, False)])
def test_plan_sizes(R, hi, tree):
    rng = random.Random(R)
    check_plan([rng.randint(0, 700) for _ in range(R)], [rng.randint(0, hi) for _ in range(R - 1)] + [hi], 16, tree, seed=R)


def test_plan_without_requests_or_rows():
    from mlir_air_b200 import ops
    ws = ops.RequestWorkspace()
    z = i32([])
    p = ops.page_plan(z, z, torch.zeros((0, 4), dtype=torch.int32, device="cuda"), i32([0, 1]), i32([2]), 16, 3, ws)
    assert p.q_start.tolist() == [0] and p.slots.tolist() == [-1] * 3
    check_plan([5, 16], [0, 0], 16, False)
    ws.check()


@pytest.mark.parametrize("what", ["pages", "rows", "width", "tree", "negative", "count"])
def test_a_step_that_does_not_fit_changes_nothing(what):
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    ws = ops.RequestWorkspace()
    table, used = make_table([20, 40], 16, 0, width=8)
    lens, new, T, count, parents = [20, 40], [30, 5], 40, [10], None
    if what == "pages":
        count = [1]
    elif what == "rows":
        T = 34
    elif what == "width":
        new, T = [109, 5], 200
    elif what == "tree":
        new, T, parents = [65, 5], 80, i32([-1] * 80)
    elif what == "negative":
        new = [30, -1]
    else:
        count = [99]
    before, free = table.clone(), i32([used + i for i in range(12)])
    c = i32(count)
    p = ops.page_plan(i32(lens), i32(new), table, free, c, 16, T, ws, parents=parents)
    assert p.q_start.tolist() == [0, 0, 0] and p.slots.tolist() == [-1] * T and p.positions.tolist() == [0] * T
    assert torch.equal(table, before) and c.tolist() == count
    with pytest.raises(AwqBackendError, match="not enough free pages" if what == "pages" else "beyond the batch"):
        ws.check()
    ops.page_plan(i32(lens), i32([1, 1]), table, free, i32([10]), 16, 4, ws)
    ws.check()


def test_plan_reports_parents_and_pages_it_cannot_use():
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    ws = ops.RequestWorkspace()
    for parents in ([0, 0, 1], [-1, 2, 0], [-2, 0, 0], [-1, 0, 9]):
        table = i32([[0, -1]])
        p = ops.page_plan(i32([3]), i32([3]), table, i32([1, 2]), i32([2]), 16, 3, ws, parents=i32(parents))
        assert p.slots.tolist() == [3, 4, 5]
        with pytest.raises(AwqBackendError, match="parent"):
            ws.check()
    for page in (-1, 2 ** 27, 2 ** 31 - 1):  # 2^27 pages of 16 have no int32 slots
        p = ops.page_plan(i32([0]), i32([3]), i32([[-1, -1]]), i32([page, page]), i32([2]), 16, 3, ws)
        assert p.slots.tolist() == [-1] * 3
        with pytest.raises(AwqBackendError, match="page outside"):
            ws.check()


def test_lengths_near_the_end_of_32_bits():
    """A table as wide as slots can be numbered, pages whose size is no power of two, a request that ends in its last page."""
    from mlir_air_b200 import ops
    page, width, ws = 1000, 2147483, ops.RequestWorkspace()
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    table[0, -1], table[1, 0] = 7, 3
    lens, new, stack, count = i32([2147482990, 1999]), i32([9, 3]), i32([5, 4, 6, -5, -5, -5]), i32([3])
    table[1, 1] = 8
    p = ops.page_plan(lens, new, table, stack, count, page, 12, ws)
    ws.check()
    assert p.q_start.tolist() == [0, 9, 12] and count.tolist() == [2] and int(table[1, 2]) == 6
    assert p.slots.tolist() == [7990 + j for j in range(9)] + [8999, 6000, 6001]
    assert p.positions.tolist() == [2147482990 + j for j in range(9)] + [1999, 2000, 2001]
    kv = torch.zeros((1, 2, 10, page, 1, 16), dtype=BF, device="cuda")
    kv[0, 0, 7, 990:999, 0, 0] = torch.arange(9, device="cuda")
    ops.page_keep(kv, table, lens, p.q_start, i32([3, 1]), stack, count, ws, path=i32([2, 5, 8] + [0] * 6 + [0, 0, 0]))
    ws.check()
    assert lens.tolist() == [2147482993, 2000] and count.tolist() == [3] and stack.tolist() == [5, 4, 6, -5, -5, -5]
    assert kv[0, 0, 7, 990:993, 0, 0].tolist() == [2, 5, 8]
    ops.page_keep(kv, table, lens, i32([0, 0, 0]), i32([0, -1]), stack, count, ws)
    ws.check()
    assert lens.tolist() == [2147482993, 0] and count.tolist() == [5] and stack.tolist() == [5, 4, 6, 3, 8, -5]


# ---- rope_append --------------------------------------------------------------------------------------------------
def rotate(x, row):
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half].float(), x[..., half:].float(), row[:, None, :half].float(), row[:, None, half:].float()
    return torch.cat([a * c - b * s, a * s + b * c], -1).to(x.dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("H,kv,D", [(1, 1, 64), (8, 2, 128), (6, 6, 80), (5, 1, 256), (40, 8, 16)])
@pytest.mark.parametrize("T", [1, 7, 130])
def test_append(dtype, H, kv, D, T):
    from mlir_air_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(T)
    page, pages, P = 16, 20, 500
    qkv = torch.randn((T, (H + 2 * kv) * D), device="cuda", generator=gen).to(dtype)
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([H * D, kv * D, kv * D], 1))
    lut = torch.randn((P, D), device="cuda", generator=gen).to(BF)
    slots = torch.randperm(page * pages, device="cuda", generator=gen)[:T].to(torch.int32)
    slots[T // 2] = -1 if T > 1 else slots[0]
    pos = torch.randint(0, P, (T,), device="cuda", generator=gen).to(torch.int32)
    kc, vc = (torch.full((pages, page, kv, D), 9.0, device="cuda").to(dtype) for _ in range(2))
    want_k, want_v = kc.clone().flatten(0, 1), vc.clone().flatten(0, 1)
    on = slots >= 0
    want_k[slots[on].long()] = rotate(k, lut[pos.long()])[on]
    want_v[slots[on].long()] = v[on]
    want_q = torch.where(on[:, None, None], rotate(q, lut[pos.long()]), q)
    out = torch.full((T, H, D), 5.0, device="cuda").to(dtype)
    ws = ops.RequestWorkspace()
    before = qkv.clone()
    ops.rope_append(q, k, v, lut, pos, slots, ops.KVCache(kc, vc), ws, q_out=out)
    assert torch.equal(qkv, before)
    assert torch.equal(out[on], want_q[on]) and bool((out[~on] == 5).all())
    assert torch.equal(kc.flatten(0, 1), want_k) and torch.equal(vc.flatten(0, 1), want_v)
    # in place, into a cache with heads in front of slots
    k2, v2 = (torch.full((pages, kv, page, D), 9.0, device="cuda").to(dtype).transpose(1, 2) for _ in range(2))
    ops.rope_append(q, k, v, lut, pos, slots, ops.KVCache(k2, v2), ws)
    assert torch.equal(q, want_q) and torch.equal(k2.flatten(0, 1), want_k) and torch.equal(v2.flatten(0, 1), want_v)
    ws.check()


def test_append_agrees_with_rope_halfsplit():
    from mlir_air_b200 import ops
    T, H, D = 33, 8, 128
    x = torch.randn((T, H * D), device="cuda").to(BF)
    lut = torch.randn((T, D), device="cuda").to(BF)
    cache = ops.KVCache(*torch.zeros((2, 4, 16, 2, D), dtype=BF, device="cuda"))
    kv = torch.randn((T, 2, D), device="cuda").to(BF)
    at = torch.arange(T, dtype=torch.int32, device="cuda")
    got = ops.rope_append(x.unflatten(1, (H, D)), kv, kv, lut, at, at, cache, ops.RequestWorkspace(), q_out=torch.empty((T, H, D), dtype=BF, device="cuda"))
    assert torch.equal(got.flatten(1), ops.rope_halfsplit(x.clone(), lut, H, D))
    assert torch.equal(cache.k.flatten(0, 1)[:T].flatten(1), ops.rope_halfsplit(kv.flatten(1).clone(), lut, 2, D))


def test_of_rows_that_name_one_slot_the_last_stays():
    from mlir_air_b200 import ops
    T, D = 700, 64
    gen = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn((T, 2, D), device="cuda", generator=gen).to(BF) for _ in range(2))
    slots = torch.randint(0, 40, (T,), device="cuda", generator=gen).to(torch.int32)
    lut = torch.cat([torch.ones(1, D // 2), torch.zeros(1, D // 2)], 1).to(BF).cuda()
    cache = ops.KVCache(*torch.zeros((2, 3, 16, 2, D), dtype=BF, device="cuda"))
    ws = ops.RequestWorkspace()
    ops.rope_append(torch.zeros((T, 2, D), dtype=BF, device="cuda"), k, v, lut, torch.zeros_like(slots), slots, cache, ws)
    ws.check()
    want = {int(s): t for t, s in enumerate(slots.tolist())}
    for s, t in want.items():
        assert torch.equal(cache.k[s // 16, s % 16], k[t]) and torch.equal(cache.v[s // 16, s % 16], v[t])


def test_append_reports_slots_and_positions():
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    D = 64
    cache = ops.KVCache(*torch.zeros((2, 3, 16, 2, D), dtype=BF, device="cuda"))
    ws = ops.RequestWorkspace()
    x = torch.ones((2, 2, D), dtype=BF, device="cuda")
    lut = torch.ones((10, D), dtype=BF, device="cuda")
    for slots, pos in (([48, 1], [0, 0]), ([-2, 1], [0, 0]), ([0, 1], [10, 0]), ([0, 1], [-1, 0]), ([2 ** 31 - 1, 1], [0, 0])):
        cache.k.zero_()
        out = torch.zeros_like(x)
        ops.rope_append(x, x, x, lut, i32(pos), i32(slots), cache, ws, q_out=out)
        with pytest.raises(AwqBackendError, match="slot outside"):
            ws.check()
        assert bool((out[0] == 0).all()) and bool((out[1] != 0).any()) and float(cache.k.abs().sum(dtype=torch.float32)) == 2 * float(out[1].abs().sum(dtype=torch.float32)) / 2
    with pytest.raises(AwqBackendError):
        ops.rope_append(x, x[:1], x, lut, i32([0, 0]), i32([0, 1]), cache, ws)
    with pytest.raises(AwqBackendError):
        ops.rope_append(x, x, x, lut[:, :32], i32([0, 0]), i32([0, 1]), cache, ws)
    with pytest.raises(AwqBackendError):
        ops.rope_append(x, x, x, lut, i32([0]), i32([0, 1]), cache, ws)
    with pytest.raises(AwqBackendError):
        ops.rope_append(x.half(), x, x, lut, i32([0, 0]), i32([0, 1]), cache, ws)


def test_a_row_that_is_left_out_takes_no_slot_from_others():
    """Of two rows that name one slot the last that has a position stays there."""
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    D = 64
    gen = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn((4, 2, D), device="cuda", generator=gen).to(BF) for _ in range(2))
    lut = torch.cat([torch.ones(10, D // 2), torch.zeros(10, D // 2)], 1).to(BF).cuda()
    for bad in (10, -1, 2 ** 31 - 1):
        cache, ws = ops.KVCache(*torch.zeros((2, 3, 16, 2, D), dtype=BF, device="cuda")), ops.RequestWorkspace()
        ops.rope_append(torch.zeros((4, 2, D), dtype=BF, device="cuda"), k, v, lut, i32([0, 1, 2, bad]), i32([5, 7, 5, 5]), cache, ws)
        with pytest.raises(AwqBackendError, match="slot outside"):
            ws.check()
        assert torch.equal(cache.k[0, 5], k[2]) and torch.equal(cache.v[0, 5], v[2]) and torch.equal(cache.k[0, 7], k[1])


# ---- page_keep ----------------------------------------------------------------------------------------------------
def keep_ref(kv, table, lens, new, kept, path, free, page):
    """The definition on a clone of kv and host lists: (kv, lens, free)."""
    kv, lens, st = kv.clone(), list(lens), starts(new)
    old = kv.clone()
    free = list(free)
    for r, n in enumerate(new):
        slot = lambda p: (table[r][p // page], p % page)  # noqa: B023, E731
        k = max(kept[r], 0)
        for i in range(k):
            a, b = slot(lens[r] + (path[st[r] + i] if path is not None else i)), slot(lens[r] + i)
            kv[:, :, b[0], b[1]] = old[:, :, a[0], a[1]]
        after = 0 if kept[r] < 0 else lens[r] + k
        free += [table[r][b] for b in range(-(-after // page), -(-(lens[r] + n) // page))]
        lens[r] = after
    return kv, lens, free


@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("layers,heads,D", [(1, 1, 64), (3, 4, 128), (2, 12, 80)])
@pytest.mark.parametrize("with_path", [True, False])
def test_keep(page, layers, heads, D, with_path):
    from mlir_air_b200 import ops
    rng = random.Random(page)
    lens, new = [0, 3, 16, 40, 9, 7, 31, 100], [5, 64, 1, 33, 0, 8, 64, 20]
    kept = [5, 20, 0, 33, 0, -1, 64, 1]
    path = [x for n, k in zip(new, kept) for x in sorted(rng.sample(range(n), max(k, 0))) + [77] * (n - max(k, 0))] if with_path else None
    table, used = make_table([l + n for l, n in zip(lens, new)], page, 1, extra=3)
    kv = torch.randn((layers, 2, used, page, heads, D), device="cuda").to(BF)
    free = [1, 2, 3]
    want = keep_ref(kv, table.tolist(), lens, new, kept, path, free, page)
    stack = i32(free + [-5] * (used - 3))
    lens_t, count = i32(lens), i32([3])
    ws = ops.RequestWorkspace()
    ops.page_keep(kv, table, lens_t, i32(starts(new)), i32(kept), stack, count, ws, path=None if path is None else i32(path))
    ws.check()
    assert torch.equal(kv, want[0]) and lens_t.tolist() == want[1]
    assert count.tolist() == [len(want[2])] and stack.tolist()[:len(want[2])] == want[2] and stack.tolist()[len(want[2]):] == [-5] * (used - len(want[2]))


def test_keep_of_many_requests():
    from mlir_air_b200 import ops
    rng = random.Random(0)
    R = 4096
    lens, new = [rng.randint(0, 40) for _ in range(R)], [rng.randint(0, 4) for _ in range(R)]
    kept = [rng.randint(-1, n) for n in new]
    path = [x for n, k in zip(new, kept) for x in sorted(rng.sample(range(n), max(k, 0))) + [0] * (n - max(k, 0))]
    table, used = make_table([l + n for l, n in zip(lens, new)], 16, 1)
    kv = torch.randn((1, 2, used, 16, 1, 16), device="cuda").to(FP)
    out_lens, out_count, stack = i32([0] * R), i32([0]), i32([-5] * used)
    ws = ops.RequestWorkspace()
    args = (table, i32(lens), i32(starts(new)), i32(kept), stack, i32([0]), ws)
    # (without a reference in 64 bits per row: the moves are checked by test_keep, here the lengths and the stack)
    ops.page_keep(kv, *args, path=i32(path), lens_out=out_lens, free_count_out=out_count)
    ws.check()
    host, want_free = table.tolist(), []
    for r in range(R):
        after = 0 if kept[r] < 0 else lens[r] + kept[r]
        want_free += host[r][-(-after // 16):-(-(lens[r] + new[r]) // 16)]
        assert out_lens[r] == after if r % 97 == 0 else True
    assert out_lens.tolist() == [0 if k < 0 else l + k for l, k in zip(lens, kept)]
    assert out_count.tolist() == [len(want_free)] and stack.tolist()[:len(want_free)] == want_free
    assert args[1].tolist() == lens and args[5].tolist() == [0]


def test_keep_reports_what_does_not_fit():
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    ws = ops.RequestWorkspace()
    lens, new = [10, 20], [8, 4]
    for kept, path in (([9, 1], None), ([-2, 1], None), ([2, 1], [3, 3]), ([2, 1], [4, 3]), ([1, 1], [8]), ([1, 1], [-1])):
        table, used = make_table([18, 24], 16, 0)
        kv = torch.randn((2, 2, used, 16, 2, 64), device="cuda").to(BF)
        before = kv.clone()
        full = None if path is None else i32(path + [0] * (8 - len(path)) + [0, 1, 2, 3])
        lens_t = i32(lens)
        ops.page_keep(kv, table, lens_t, i32([0, 8, 12]), i32(kept), i32([0] * used), i32([0]), ws, path=full)
        with pytest.raises(AwqBackendError, match="count or path"):
            ws.check()
        assert torch.equal(kv, before) and lens_t.tolist() == [10, 21]
    # pages outside the cache are not touched
    table, used = make_table([18, 24], 16, 0)
    kv = torch.randn((2, 2, used, 16, 2, 64), device="cuda").to(BF)
    before = kv.clone()
    table[0, 0] = used
    ops.page_keep(kv, table, i32(lens), i32([0, 8, 12]), i32([2, 1]), i32([0] * used), i32([0]), ws, path=i32([3, 4] + [0] * 6 + [0, 1, 2, 3]))
    with pytest.raises(AwqBackendError, match="page outside"):
        ws.check()
    assert torch.equal(kv, before)
    with pytest.raises(AwqBackendError):
        ops.page_keep(kv[0], table, i32(lens), i32([0, 8, 12]), i32([2, 1]), i32([0] * used), i32([0]), ws)
    with pytest.raises(AwqBackendError):
        ops.page_keep(kv, table, i32(lens), i32([0, 8]), i32([2, 1]), i32([0] * used), i32([0]), ws)


@pytest.mark.parametrize("what", ["short path", "starts beyond the path", "start below zero", "start behind the next", "length beyond the table", "length below zero"])
@pytest.mark.parametrize("ends", [False, True])
def test_a_request_whose_range_does_not_fit_keeps_its_state(what, ends):
    """Its length, its rows and its pages stay as they are, also if it was to end; the other requests are served."""
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    ws = ops.RequestWorkspace()
    lens, new, start = [10, 40, 17], [8, 4, 20], [0, 8, 12, 32]
    kept, bad, path = [2, 1, 5], [2], [0, 3] + [0] * 6 + [2, 0, 0, 0] + [1, 4, 5, 8, 9] + [0] * 15
    table, used = make_table([18, 44, 37], 16, 0, width=4)
    if what == "short path":
        path = path[:17]
    elif what == "starts beyond the path":
        start[2:], bad = [40, 60], [1, 2]
    elif what == "start below zero":
        start[0], bad = -1, [0]
    elif what == "start behind the next":
        start[1], bad = 20, [0, 1]
        start[0] = 21
    elif what == "length beyond the table":
        lens[2] = 64
    else:
        lens[1], bad = -3, [1]
    if ends:
        kept = [-1 if r in bad else k for r, k in enumerate(kept)]
    kv = torch.randn((2, 2, used, 16, 2, 64), device="cuda").to(BF)
    before, stack, count, lens_t = kv.clone(), i32([-5] * used), i32([0]), i32(lens)
    ops.page_keep(kv, table, lens_t, i32(start), i32(kept), stack, count, ws, path=i32(path))
    with pytest.raises(AwqBackendError, match="count or path"):
        ws.check()
    assert lens_t.tolist() == [l if r in bad else l + kept[r] for r, l in enumerate(lens)]
    host, free, want = table.tolist(), [], before.clone()
    for r in range(3):
        if r in bad:
            continue
        slot = lambda p: (host[r][p // 16], p % 16)  # noqa: B023, E731
        for i in range(kept[r]):
            a, b = slot(lens[r] + path[start[r] + i]), slot(lens[r] + i)
            want[:, :, b[0], b[1]] = before[:, :, a[0], a[1]]
        free += host[r][-(-(lens[r] + kept[r]) // 16):-(-(lens[r] + start[r + 1] - start[r]) // 16)]
    assert torch.equal(kv, want)
    assert count.tolist() == [len(free)] and stack.tolist() == free + [-5] * (used - len(free))
    ops.page_keep(kv, table, i32([10, 40, 17]), i32([0, 0, 0, 0]), i32([0, 0, 0]), stack, count, ws)
    ws.check()


# ---- together -----------------------------------------------------------------------------------------------------
def test_steps_of_a_serving_loop():
    """Prompts, drafted trees, acceptance, requests that end and new ones in their place: after every step the cache holds, for
    every request, exactly its tokens' K and V, no page belongs to two requests, and attention over the pages equals attention
    over the tokens that a plain list remembers."""
    from mlir_air_b200 import ops
    rng = random.Random(11)
    R, page, pages, H, kv, D, layers = 5, 16, 60, 8, 2, 64, 2
    cache = torch.full((layers, 2, pages, page, kv, D), float("nan"), device="cuda").to(BF)
    handles = [ops.KVCache(cache[i, 0], cache[i, 1]) for i in range(layers)]
    lens, table, stack, count = i32([0] * R), torch.full((R, 30), -1, dtype=torch.int32, device="cuda"), i32(list(range(pages))), i32([pages])
    lut = torch.cat([torch.ones(1000, D // 2), torch.zeros(1000, D // 2)], 1).to(BF).cuda()  # no rotation: K as it came
    ws = ops.RequestWorkspace()
    ref = [[torch.zeros((0, 2, kv, D), dtype=BF, device="cuda") for _ in range(R)] for _ in range(layers)]
    for step in range(12):
        tree = step % 3 != 0
        new = [rng.randint(1, 20) if tree else rng.randint(0, 50) if len(ref[0][r]) == 0 else rng.randint(0, 2) for r in range(R)]
        T = sum(new) + 3
        st = starts(new)
        parents = [rng.randint(max(-1, j - 3), j - 1) for n in new for j in range(n)]
        plan = ops.page_plan(lens, i32(new), table, stack, count, page, T, ws, parents=i32(parents + [0] * 3) if tree else None)
        rows = []
        for i in range(layers):
            q, k, v = (torch.randn((T, n, D), device="cuda").to(BF) for n in (H, kv, kv))
            ops.rope_append(q, k, v, lut, plan.positions, plan.slots, handles[i], ws)
            got = ops.tree_attention(q, handles[i], table, lens, plan.q_start, ws, mask=plan.mask)
            rows.append(torch.stack([k, v], 1))
            for r in range(R):
                for j in range(new[r]):
                    if tree:
                        seen, p = [j], j
                        while parents[st[r] + p] >= 0:
                            p = parents[st[r] + p]
                            seen.append(p)
                        seen = sorted(seen)
                    else:
                        seen = list(range(j + 1))
                    ctx = torch.cat([ref[i][r], rows[i][st[r]:st[r + 1]][seen]]).double()
                    for h in range(H):
                        w = torch.softmax(ctx[:, 0, h * kv // H] @ q[st[r] + j, h].double() * D ** -0.5, 0)
                        want = w @ ctx[:, 1, h * kv // H]
                        mag = w @ ctx[:, 1, h * kv // H].abs()
                        assert bool(((got[st[r] + j, h].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-4) * mag).all())
        kept, path = [], []
        for r in range(R):
            if step % 4 == 3 and r == step % R:
                kept.append(-1)
                path += [0] * new[r]
                continue
            k = rng.randint(0, min(new[r], 6)) if tree else new[r]
            p = sorted(rng.sample(range(new[r]), k)) if tree else list(range(k))
            kept.append(k)
            path += p + [0] * (new[r] - k)
        if not tree:
            path = None
        ops.page_keep(cache, table, lens, plan.q_start, i32(kept), stack, count, ws, path=None if path is None else i32(path + [0] * 3))
        ws.check()
        host, own = table.tolist(), set(stack[:int(count)].tolist())
        assert len(own) == int(count)
        for r in range(R):
            for i in range(layers):
                new_rows = rows[i][st[r]:st[r + 1]]
                idx = list(range(max(kept[r], 0))) if path is None else path[st[r]:st[r] + max(kept[r], 0)]
                ref[i][r] = ref[i][r][:0] if kept[r] < 0 else torch.cat([ref[i][r], new_rows[idx]])
            n = len(ref[0][r])
            assert int(lens[r]) == n
            mine = host[r][:-(-n // page)]
            assert not own & set(mine) and len(set(mine)) == len(mine)
            own |= set(mine)
            for i in range(layers):
                for p in range(n):
                    assert torch.equal(cache[i, :, host[r][p // page], p % page], ref[i][r][p])
        assert own == set(range(pages))
