"""lora against 64 bits: ranks, orders of rows, formats of the base, what lies behind an adapter's rank."""
import pytest
import torch

from request_util import i32, lora_ref

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def make(T, K, N, n, rank_max, ranks, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    A, B = (rnd(n, rank_max, K) * K ** -0.5).to(BF), (rnd(n, N, rank_max) * 0.3).to(BF)
    for a, r in enumerate(ranks or []):  # behind an adapter's rank: not read
        A[a, r:] = float("nan")
        B[a, :, r:] = float("nan")
    return rnd(T, K).to(BF), A, B, torch.rand(n, device="cuda", generator=gen) * 2 - 0.5, None if ranks is None else i32(ranks), rnd(T, N)


def check(T, K, N, idx, ranks, rank_max=16, n=None, base_f32=True, residual=False, seed=0):
    from mlir_air_b200 import ops
    n = n or (len(ranks) if ranks is not None else max(idx) + 1)
    x, A, B, s, rk, base = make(T, K, N, n, rank_max, ranks, seed)
    base = base if base_f32 else base.to(BF)
    res = torch.randn((T, N), device="cuda").to(BF) if residual else None
    ws = ops.RequestWorkspace()
    out = ops.lora(x, ops.LoraAdapters(A, B, s, rk), i32(idx), base, ws, residual=res)
    ws.check()
    ref, tol = lora_ref(x, A, B, s, ranks, torch.tensor(idx), base, res)
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), f"{int((err > tol).sum())} of {err.numel()} values are off, at most {float((err / tol).max()):.2f} times"
    return out


@pytest.mark.parametrize("T", [1, 2, 5, 16, 17, 64, 65, 200])
@pytest.mark.parametrize("base_f32,residual", [(True, False), (False, True)])
def test_rows(T, base_f32, residual):
    check(T, 512, 384, [(t * 7) % 5 - 1 for t in range(T)], [16, 1, 9, 16], base_f32=base_f32, residual=residual)


@pytest.mark.parametrize("rank_max", [8, 16, 24, 40, 64, 72, 128])
@pytest.mark.parametrize("T", [1, 9, 80])
def test_ranks(rank_max, T):
    check(T, 640, 264, [t % 4 for t in range(T)], [rank_max, rank_max - 1, 1, 0], rank_max)
    check(T, 640, 264, [t % 2 for t in range(T)], None, rank_max)


@pytest.mark.parametrize("K,N", [(8, 8), (16, 8), (72, 1000), (1000, 72), (4096, 40), (40, 4096), (2056, 2056), (11008, 136)])
@pytest.mark.parametrize("T", [1, 37, 70])
def test_sizes(K, N, T):
    check(T, K, N, [0 if t % 3 else 1 for t in range(T)], [12, 16], seed=K)


def test_orders_of_rows():
    """Sorted, reversed, mixed, one adapter for all, one each, none at all: a row's result is its own."""
    T = 150
    rows = {}
    for name, idx in (("runs", [t // 50 for t in range(T)]), ("reversed", [2 - t // 50 for t in range(T)]), ("mixed", [(t * t) % 3 for t in range(T)]),
                      ("one", [1] * T), ("none", [-1] * T)):
        out = check(T, 256, 128, idx, [16, 8, 3], n=3)
        for t, a in enumerate(idx):
            if (t, a) in rows:
                assert torch.equal(out[t], rows[t, a]), (name, t, a)
            rows[t, a] = out[t]
    check(100, 256, 128, list(range(100)), None)


def test_many_rows_and_adapters():
    check(3000, 256, 136, [(t // 211) % 9 - 1 for t in range(3000)], [64, 5, 33, 64, 8, 17, 1, 40], 64, base_f32=False)
    check(700, 136, 256, [(t * 31) % 300 for t in range(700)], None, 8)


def test_in_place_and_strides():
    from mlir_air_b200 import ops
    x, A, B, s, rk, base = make(30, 512, 256, 3, 16, [16, 4, 9])
    idx, ws, ad = i32([t % 4 - 1 for t in range(30)]), ops.RequestWorkspace(), ops.LoraAdapters(A, B, s, rk)
    b16 = base.to(BF)
    want = ops.lora(x, ad, idx, b16, ws)
    wide = torch.full((30, 520 + 8), float("nan"), device="cuda").to(BF)
    wide[:, 8:520] = x
    assert torch.equal(ops.lora(wide[:, 8:520], ad, idx, b16, ws), want)
    got = ops.lora(x, ad, idx, b16, ws, out=b16)
    assert got is b16 and torch.equal(got, want)
    none = idx < 0
    assert torch.equal(want[none], base.to(BF)[none])
    ws.check()


@pytest.mark.parametrize("T", [5, 140])
def test_the_residual_may_be_overwritten(T):
    from mlir_air_b200 import ops
    x, A, B, s, rk, base = make(T, 512, 512, 3, 16, [16, 3, 8])
    res, ws = torch.randn((T, 512), device="cuda").to(BF), ops.RequestWorkspace()
    args = (x, ops.LoraAdapters(A, B, s, rk), i32([t % 4 - 1 for t in range(T)]), base, ws)
    want = ops.lora(*args, residual=res)
    assert ops.lora(*args, residual=res, out=res) is res and torch.equal(res, want)
    with pytest.raises(Exception, match="overlap"):
        ops.lora(*args, out=x)
    ws.check()


def test_beside_an_int4_projection():
    """gemv's f32 sums, then the adapters and the residual with one rounding: what a decode layer with adapters computes."""
    import numpy as np
    from gpu_util import dev_weight, randn_bf16, synth_awq, to_dev
    from mlir_air_b200 import ops
    K, N, T = 512, 768, 6
    q = synth_awq(K, N, seed=4)
    w, wws, ws = dev_weight(*q), ops.Workspace(K, N), ops.RequestWorkspace()
    _, A, B, s, rk, _ = make(T, K, N, 3, 16, [16, 2, 7])
    x, res, idx = to_dev(randn_bf16((T, K), 1)), to_dev(randn_bf16((T, N), 2)), i32([2, -1, 0, 0, 1, 2])
    base = ops.gemv(x, w, wws, f32_out=True)
    got = ops.lora(x, ops.LoraAdapters(A, B, s, rk), idx, base, ws, residual=res)
    wws.check()
    ws.check()
    # the weights as the projection multiplies them: (q - z) s, not rounded to bf16 as `dequant` does
    steps = ops.dequant(ops.AwqWeight(w.qweight, w.qzeros, torch.ones_like(w.scales))).double()
    wide = steps * w.scales.double().repeat_interleave(128, 0)
    full = x.double() @ wide
    ref, tol = lora_ref(x, A, B, s, [16, 2, 7], idx.cpu(), full, res)
    # the projection's own f32 sum and its 2^-20 hand-over, on top
    tol = tol + 2.0 ** -18 + 2.0 ** -20 * (x.double().abs() @ wide.abs())
    assert bool(((got.double() - ref).abs() <= tol).all())
    assert np.isfinite(got.float().cpu().numpy()).all()


def test_adapters_that_do_not_exist_are_reported():
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    x, A, B, s, rk, base = make(20, 64, 64, 2, 8, [8, 3])
    ad, ws = ops.LoraAdapters(A, B, s, rk), ops.RequestWorkspace()
    good = ops.lora(x, ad, i32([0, 1] * 10), base, ws)
    ws.check()
    for bad in (2, 2 ** 31 - 1):
        out = ops.lora(x, ad, i32([0, 1] * 9 + [0, bad]), base, ws)
        assert torch.equal(out[:19], good[:19]) and torch.equal(out[19], base[19].to(BF))
        with pytest.raises(AwqBackendError, match="adapter"):
            ws.check()
    out = ops.lora(x, ad, i32([0, 1] * 9 + [0, -2 ** 31]), base, ws)
    ws.check()
    assert torch.equal(out[19], base[19].to(BF))
    # ranks beyond the storage are cut to it
    assert torch.equal(ops.lora(x, ops.LoraAdapters(A[:1], B[:1], s[:1], i32([99])), i32([0] * 20), base, ws),
                       ops.lora(x, ops.LoraAdapters(A[:1], B[:1], s[:1]), i32([0] * 20), base, ws))
    empty = ops.lora(x[:0], ad, i32([]), base[:0], ws)
    assert empty.shape == (0, 64)


def test_arguments_that_do_not_fit_are_refused():
    from mlir_air_b200 import ops
    from mlir_air_b200._lib import AwqBackendError
    x, A, B, s, rk, base = make(20, 64, 64, 2, 8, [8, 3])
    ad, ws, idx = ops.LoraAdapters(A, B, s, rk), ops.RequestWorkspace(), i32([0] * 20)
    for args in ((x[:, :32], idx, base), (x.half(), idx, base), (x, idx.long(), base), (x, idx[:-1], base), (x, idx, base.half()),
                 (x, idx, base[:, :32]), (x, idx, base[:-1]), (x.cpu(), idx, base)):
        with pytest.raises(AwqBackendError):
            ops.lora(args[0], ad, args[1], args[2], ws)
    with pytest.raises(AwqBackendError):
        ops.lora(x, ad, idx, base, ws, out=base)
    with pytest.raises(AwqBackendError):
        ops.lora(x, ad, idx, base, ws, residual=base)
    for bad in ((A[:, :5], B[..., :5], s, None), (A, B[:1], s, rk), (A, B, s[:1], rk), (A, B, s, rk[:1]), (A.float(), B, s, rk), (A, B, s.double(), rk),
                (A[..., :60], B, s, rk), (A.cpu(), B, s, rk)):
        with pytest.raises(AwqBackendError):
            ops.LoraAdapters(*bad)


def test_streams_and_graphs():
    from mlir_air_b200 import ops
    x, A, B, s, rk, base = make(70, 512, 256, 3, 16, [16, 4, 9])
    ad, ws, ws2 = ops.LoraAdapters(A, B, s, rk), ops.RequestWorkspace(), ops.RequestWorkspace()
    idx = i32([t % 4 - 1 for t in range(70)])
    want = ops.lora(x, ad, idx, base, ws)
    torch.cuda.synchronize()
    side, out = torch.cuda.Stream(), torch.empty_like(want)
    with torch.cuda.stream(side):
        ops.lora(x, ad, idx, base, ws2, out=out)
    again = ops.lora(x, ad, idx, base, ws)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.lora(x, ad, idx, base, ws, out=out)
    idx2 = i32([(t // 9) % 4 - 1 for t in range(70)])
    want2 = ops.lora(x, ad, idx2, base, ws)
    idx.copy_(idx2)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want2)


@pytest.mark.parametrize("T", [1, 20, 128, 200])
@pytest.mark.parametrize("rank_max,ranks", [(8, [1, 2, 8]), (16, [1, 3, 5]), (64, [1, 2, 33])])
def test_infinite_and_missing_numbers_stay_what_they_are(T, rank_max, ranks):
    """An infinite x gives what the formula gives, infinities where they do not meet their opposites; NaN gives NaN; other rows are as they were."""
    from mlir_air_b200 import ops
    x, A, B, s, rk, base = make(T, 512, 264, 3, rank_max, ranks)
    idx, ws, ad = i32([t % 4 - 1 for t in range(T)]), ops.RequestWorkspace(), ops.LoraAdapters(A, B, s, rk)
    if T == 1:
        idx[0] = 0
    was = ops.lora(x, ad, idx, base, ws)
    rows = list(range(0, T, 3))
    for i, t in enumerate(rows):
        x[t, (37 * t) % 512] = (float("inf"), -float("inf"), float("nan"))[i % 3]
    got = ops.lora(x, ad, idx, base, ws)
    ws.check()
    want, _ = lora_ref(x, A, B, s, ranks, idx.cpu(), base)
    odd = torch.zeros(T, dtype=torch.bool, device="cuda")
    odd[rows] = True
    odd &= idx >= 0
    assert torch.equal(got[~odd], was[~odd])
    same = lambda t: t[odd].double().nan_to_num(nan=7.0, posinf=8.0, neginf=9.0)  # noqa: E731
    assert torch.equal(same(got), same(want)) and bool(torch.isinf(got).any())


@pytest.mark.parametrize("T", [3, 150])
def test_a_sum_between_the_largest_numbers_of_two_formats(T):
    """x A^T beyond bf16's largest number, but not f32's: the product with a small B is finite."""
    from mlir_air_b200 import ops
    x, A, B = torch.zeros((T, 64), dtype=BF, device="cuda"), torch.zeros((1, 8, 64), dtype=BF, device="cuda"), torch.zeros((1, 64, 8), dtype=BF, device="cuda")
    x[:, 3], x[:, 9], A[0, 0, 3], A[0, 0, 9], B[0, :, 0] = torch.finfo(BF).max, 1.5 * 2.0 ** 119, 1, 1, 2.0 ** -10
    ws, base = ops.RequestWorkspace(), torch.zeros((T, 64), device="cuda")
    args = (x, A, B, torch.ones(1, device="cuda"), None)
    got = ops.lora(x, ops.LoraAdapters(*args[1:4]), i32([0] * T), base, ws)
    ws.check()
    ref, tol = lora_ref(*args, torch.zeros(T, dtype=torch.int64), base)
    assert bool(torch.isfinite(ref).all()) and bool(((got.double() - ref).abs() <= tol).all())
