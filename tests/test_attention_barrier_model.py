"""The barriers of tree_attention's tcgen05 kernel, modelled on the host: its warp roles as coroutines under random schedules, with
waits that, like an mbarrier's, tell a phase from its neighbour only.  No schedule may deadlock, and nothing may be written while it is
still to be read: the stages of K and V, the scores, the sums, the words that say which keys there are."""
import os
import random
import re

import pytest


class Bar:
    """An mbarrier: `count` arrivals complete a phase; a wait on parity p passes unless the current phase has that parity."""

    def __init__(self, count):
        self.count, self.pending, self.phase = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def passes(self, parity):
        return self.phase % 2 != parity


def run(segments, seed, rescale=0.5, tma=False, odd=0.0, warps=1):
    """warps: the softmax warps, each on its own (1: as one role).  odd: the share of tiles whose V holds what is not finite.  The warp that brings V takes it out and raises the segment's flag; the softmax
    warps put it back where it is seen, which takes them a while, if they find the flag when the segment's sums are there."""
    rng = random.Random(seed)
    total = sum(segments)
    k_full, v_full, scored, weighed = ([Bar(n), Bar(n)] for n in (1, 1, 1, warps))
    added, q_full, q_free, summed = [Bar(1) for _ in range(4)], Bar(1), Bar(1), Bar(1)
    segment_of = [i for i, t in enumerate(segments) for _ in range(t)]
    K, V, S, valid = [None] * 2, [None] * 2, [None] * 2, [None] * 4  # what each place holds
    queue, state = [], dict(q=None, o=None, weights={}, done=0)
    flags, draw = [False] * 4, random.Random(-1 - seed)
    raised = [odd > 0 and draw.random() < odd for _ in segment_of]  # by a tile

    def clean(n):
        if raised[n]:
            flags[segment_of[n] % 4] = True

    def phase(t):
        return t >> 1 & 1

    def loader(is_v):
        """One warp for K, one for V; it waits for its own copies."""
        n = 0
        for seg, tiles in enumerate(segments):
            yield from describe(seg)
            for _ in range(tiles):
                if n > 1:
                    yield (added[(n - 2) % 4], (n - 2) >> 2 & 1) if is_v else (scored[n % 2], phase(n - 2))
                place = V if is_v else K
                assert place[n % 2] is None or place[n % 2][1] == "read", (n, is_v, place)
                place[n % 2] = (n, "loading")
                if not is_v:
                    assert valid[n % 4] is None or valid[n % 4][1] == "read"
                    valid[n % 4] = (n, "there")
                yield None
                place[n % 2] = (n, "there")
                if is_v:
                    clean(n)
                (v_full if is_v else k_full)[n % 2].arrive()
                n += 1

    found, ring = [Bar(1) for _ in range(4)], [None] * 4  # the segments' descriptions, and the roles that have read each

    def describe(seg):
        """A role's wait for a segment's description."""
        yield found[seg % 4], seg >> 2 & 1
        assert ring[seg % 4][0] == seg, "a description overwritten before a role had it"
        ring[seg % 4][1] += 1

    def q_loader():
        for seg in range(len(segments)):
            assert ring[seg % 4] is None or ring[seg % 4][1] == 3 + warps
            ring[seg % 4] = [seg, 0]
            flags[seg % 4] = False
            found[seg % 4].arrive()
            yield None
            if seg:
                yield q_free, (seg - 1) % 2
            assert state["q"] is None or state["q"][1] == "read"
            state["q"] = (seg, "loading")
            yield None
            state["q"] = (seg, "there")
            q_full.arrive()

    def tma_loader(is_v, landing):
        """One warp for K, one for V; the bytes arrive by themselves, later, while it goes on.  Some tiles of V are put right first."""
        n = 0
        for seg, tiles in enumerate(segments):
            yield from describe(seg)
            for _ in range(tiles):
                if n > 1:
                    yield (added[(n - 2) % 4], (n - 2) >> 2 & 1) if is_v else (scored[n % 2], phase(n - 2))
                place = V if is_v else K
                assert place[n % 2] is None or place[n % 2][1] == "read", (n, is_v, place)
                place[n % 2] = (n, "loading")
                if not is_v:
                    assert valid[n % 4] is None or valid[n % 4][1] == "read"
                    valid[n % 4] = (n, "there")
                if is_v and (rng.random() < 0.3 or raised[n]):
                    yield None
                    place[n % 2] = (n, "there")
                    clean(n)
                    v_full[n % 2].arrive()
                else:
                    landing.append((place, n, v_full if is_v else k_full))
                n += 1

    def memory(landing):
        while state["done"] < 2 * total:
            if landing:
                place, n, bar = landing.pop(rng.randrange(len(landing)))
                place[n % 2] = (n, "there")
                bar[n % 2].arrive()
                yield None
            else:
                yield False

    def score(n, last):
        yield k_full[n % 2], phase(n)
        assert K[n % 2] == (n, "there")
        queue.append(("score", n, last))

    def products():
        n = 0
        for seg, tiles in enumerate(segments):
            yield from describe(seg)
            yield q_full, seg % 2
            yield from score(n, tiles == 1)
            for i in range(tiles):
                if i + 1 < tiles:
                    yield from score(n + 1, i + 2 == tiles)
                yield v_full[n % 2], phase(n)
                yield weighed[n % 2], phase(n)
                assert V[n % 2] == (n, "there")
                queue.append(("add", n, i == 0, i + 1 == tiles))
                n += 1

    def tensor_cores():
        """Takes the products in the order they were issued; a commit's arrival comes a while after its product."""
        while state["done"] < 2 * total:
            if not queue:
                yield False
                continue
            op = queue.pop(0)
            n = op[1]
            yield None
            if op[0] == "score":
                assert K[n % 2] == (n, "there") and state["q"] == (segment_of[n], "there")
                assert S[n % 2] is None or S[n % 2][1] == "added", "scores over weights that are still wanted"
                yield None
                S[n % 2], K[n % 2] = (n, "scores"), (n, "read")
                scored[n % 2].arrive()
                if op[2]:
                    state["q"] = (segment_of[n], "read")
                    q_free.arrive()
            else:
                assert V[n % 2] == (n, "there") and S[n % 2] == (n, "weights")
                assert state["o"] != "busy" and (not op[2] or state["o"] is None), "sums overwritten before they were taken"
                yield None
                S[n % 2], V[n % 2] = (n, "added"), (n, "read")
                state["o"] = n
                added[n % 4].arrive()
                if op[3]:
                    summed.arrive()
            state["done"] += 1

    at, took = {}, {}  # softmax warps that have weighed a tile, or taken a segment's sums

    def softmax():
        n = 0
        for seg, tiles in enumerate(segments):
            yield from describe(seg)
            for i in range(tiles):
                yield scored[n % 2], phase(n)
                assert S[n % 2] == (n, "scores") and valid[n % 4] == (n, "there")
                yield None
                if i > 0 and rng.random() < rescale:
                    yield added[(n - 1) % 4], (n - 1) >> 2 & 1
                    assert state["o"] in (n - 1, "busy"), "sums rescaled before the last product is in them"
                    state["o"] = "busy" if warps == 1 else n - 1
                    yield None
                    state["o"] = n - 1
                assert S[n % 2] == (n, "scores") and valid[n % 4] == (n, "there")
                at[n] = at.get(n, 0) + 1
                if at[n] == warps:
                    valid[n % 4], S[n % 2] = (n, "read"), (n, "weights")
                weighed[n % 2].arrive()
                n += 1
            yield summed, seg % 2
            assert state["o"] == n - 1
            for _ in range(8 if odd else 0):  # (a warp takes its time)
                assert flags[seg % 4] == any(raised[n - tiles:n]), "a segment's flag lost, or another one's"
                yield None
            yield None
            took[seg] = took.get(seg, 0) + 1
            if took[seg] == warps:
                state["o"] = None

    landing = []
    loaders = [("k", tma_loader(0, landing)), ("v", tma_loader(1, landing)), ("memory", memory(landing))] if tma else \
        [("k", loader(0)), ("v", loader(1))]
    roles = {name: [r, None] for name, r in [("mma", products()), ("tc", tensor_cores()), ("softmax", softmax()), ("q", q_loader())] + loaders +
             [(f"softmax {i}", softmax()) for i in range(1, warps)]}
    speed = {name: rng.choice([1, 1, 3, 30]) for name in roles}  # some roles far behind the others
    idle = 0
    while roles:
        name = rng.choices(list(roles), [1.0 / speed[k] for k in roles])[0]
        role, wait = roles[name]
        if wait is not None and not wait[0].passes(wait[1]):
            idle += 1
            assert idle < 20000, f"no progress: {sorted(roles)} at {state}"
            continue
        try:
            step = next(role)
            idle = idle + 1 if step is False else 0
            assert idle < 20000, f"no progress: {sorted(roles)} at {state}"
            roles[name][1] = step or None
        except StopIteration:
            del roles[name]
    assert state["done"] == 2 * total and not queue


@pytest.mark.parametrize("tma", [False, True])
@pytest.mark.parametrize("segments", [[1], [2], [3], [1, 1, 1, 1, 1], [2, 1, 3, 1, 1, 4], [17], [5, 9, 1, 6], [40]])
def test_no_schedule_deadlocks_or_overwrites(segments, tma):
    for seed in range(60):
        run(segments, seed, rescale=(0.0, 0.5, 1.0)[seed % 3], tma=tma)


@pytest.mark.parametrize("tma", [False, True])
@pytest.mark.parametrize("segments", [[1, 1, 1, 1, 1], [5, 9, 1, 6], [2, 1, 3, 1, 1, 4], [1] * 12, [1, 1, 2] * 4, [3] * 6, [40]])
def test_every_segment_keeps_its_flag(segments, tma):
    """Values that are not finite, in some tiles: whoever raises, reads and clears the flags, a segment's is there for all its readers."""
    for seed in range(100):
        run(segments, seed, rescale=(0.0, 0.5, 1.0)[seed % 3], tma=tma, odd=(0.2, 0.5)[seed % 2], warps=(1, 4)[seed // 2 % 2])


@pytest.mark.parametrize("tma", [False, True])
@pytest.mark.parametrize("segments", [[1], [3], [1, 1, 1, 1, 1], [2, 1, 3, 1, 1, 4], [5, 9, 1, 6], [20]])
def test_softmax_warps_need_not_stay_together(segments, tma):
    for seed in range(60):
        run(segments, seed, rescale=(0.0, 0.5, 1.0)[seed % 3], tma=tma, warps=4)


def test_every_wait_between_the_roles_has_a_limit():
    """A warp whose wait gives up leaves for the kernel's end.  A barrier that it will not come to any more would hold the others for good, so
    between the first role and the end there is none: the roles wait at mbarriers, each time with a limit."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlir_air_b200", "csrc", "awq_tree_attention.cu")
    text = open(path).read()
    kernel = text[text.index("tree_attention_tiles_kernel("):text.index("tree_attention_join_kernel(")]
    roles = kernel[kernel.index("---- TMA: warp 4 K"):kernel.index("req_error(&a.header->error, REQ_ERR_TIMEOUT)")]
    assert len(re.findall(r"mbar_wait_bounded_warp\(", roles)) > 10
    assert not re.findall(r"named_bar\w*|__syncthreads\w*|bar\.sync|barrier\.|mbar_wait\(|while \(", roles)
    assert kernel.count("__syncthreads()") - kernel[:kernel.index("---- TMA: warp 4 K")].count("__syncthreads()") == 1  # where they all end


def test_a_warp_that_gave_up_waits_for_its_copies_and_products():
    """Whoever leaves early must not leave copies or products behind that still write to shared or tensor memory when the CTA gives it back: all
    that is in flight when a wait of its warp gives up is waited for, with a limit, at the kernel's end.  Which tiles that are, for any number
    of tiles issued: the last two, and all before them have been waited for already."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlir_air_b200", "csrc", "awq_tree_attention.cu")
    text = open(path).read()
    kernel = text[text.index("tree_attention_tiles_kernel("):text.index("tree_attention_join_kernel(")]
    end = kernel[kernel.index("req_error(&a.header->error, REQ_ERR_TIMEOUT)"):]
    end = end[:end.index("__syncthreads()")]
    for what in ("v_full : k_full, t", "v_landed", "dg_umma_commit(smem_u32(&sh.drained))", "smem_u32(&sh.drained), 0"):
        assert what in end, what
    assert end.count("WAIT_LIMIT_DEFAULT") == 3  # (not the call's own limit, which may be a short one)
    # K's and V's warp issue tile n once tile n - 2 has been scored or added, so that its copies have landed
    for n in range(12):
        landed = {t for t in range(n) if t + 2 < n}
        assert landed | set(range(max(n - 2, 0), n)) == set(range(n))
