"""Refusals of the operators on many requests' rows that need no GPU: bad sizes, strides, pointers and workspaces are status codes with a
message before anything touches the device."""
import ctypes

import pytest

from mlir_air_b200 import _lib

P = ctypes.c_void_p(4096)   # 16-byte aligned, never dereferenced
ODD = ctypes.c_void_p(4096 + 2)
BIG = 1 << 40


def err(rc, status=_lib.AWQ_ERR_INVALID_ARGUMENT, text=""):
    assert rc == status, (rc, _lib.last_error())
    assert _lib.last_error() and text in _lib.last_error(), _lib.last_error()


def cache(**change):
    f = dict(k=4096, v=4096, k_page_stride=16 * 256, k_slot_stride=256, k_head_stride=128, v_page_stride=16 * 256, v_slot_stride=256,
             v_head_stride=128, n_pages=10, page_size=16, n_kv_heads=2, head_dim=128, format=0)
    f.update(change)
    c = _lib.KvCacheStruct(**f)
    return ctypes.byref(c), c


BAD_CACHES = [dict(k=None), dict(v=None), dict(format=2), dict(n_pages=0), dict(page_size=0), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=100),
              dict(head_dim=272), dict(k=4098), dict(v=4104), dict(k_page_stride=12), dict(v_head_stride=-8), dict(n_pages=1 << 28)]


def test_workspace():
    lib = _lib.load()
    n = int(lib.awq_b200_request_workspace_bytes())
    assert 256 < n < 1 << 28
    err(lib.awq_b200_request_check(None, None))


def attend(c, **change):
    a = dict(q=P, qr=1024, qh=128, cache=c, table=P, stride=4, width=4, lens=P, start=P, mask=None, scale=1.0, out=P, orow=1024, oh=128, R=2, T=5,
             H=8, ws=P, nbytes=BIG, stream=None)
    a.update(change)
    return _lib.load().awq_b200_tree_attention(*a.values())


def test_tree_attention():
    c, keep = cache()
    for bad in BAD_CACHES:
        b, keep2 = cache(**bad)
        err(attend(b))
    err(attend(None))
    for bad in (dict(R=-1), dict(R=4097), dict(T=-1), dict(T=(1 << 20) + 1), dict(width=-1), dict(H=0), dict(H=7), dict(stride=3), dict(qr=1020),
                dict(oh=-8), dict(q=None), dict(out=None), dict(table=None), dict(lens=None), dict(start=None), dict(q=ODD), dict(out=ODD),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(ws=ODD)):
        err(attend(c, **bad))
    err(attend(c, ws=None), _lib.AWQ_ERR_WORKSPACE)
    err(attend(c, nbytes=1000), _lib.AWQ_ERR_WORKSPACE)
    assert attend(c, R=0) == 0 and attend(c, T=0) == 0


def append(c, **change):
    a = dict(q=P, qr=1024, qh=128, k=P, kr=256, kh=128, v=P, vr=256, vh=128, lut=P, n_pos=100, pos=P, slots=P, out=P, orow=1024, oh=128, cache=c, T=5,
             H=8, ws=P, nbytes=BIG, stream=None)
    a.update(change)
    return _lib.load().awq_b200_rope_append(*a.values())


def test_rope_append():
    c, keep = cache()
    for bad in BAD_CACHES:
        b, keep2 = cache(**bad)
        err(append(b))
    for bad in (dict(T=-1), dict(T=(1 << 20) + 1), dict(H=-1), dict(n_pos=0), dict(qr=4), dict(kh=-8), dict(vr=9), dict(orow=1), dict(q=None), dict(k=None),
                dict(v=None), dict(lut=None), dict(pos=None), dict(slots=None), dict(out=None), dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(lut=ODD),
                dict(out=ODD)):
        err(append(c, **bad))
    err(append(c, nbytes=0), _lib.AWQ_ERR_WORKSPACE)
    assert append(c, T=0) == 0


def test_cache_strides_of_zero():
    """A dimension of one may come with any stride, 0 among them; a longer one may not repeat the same values: what brings whole boxes of the
    cache would read them from elsewhere."""
    for bad in (dict(k_head_stride=0), dict(v_head_stride=0), dict(k_slot_stride=0), dict(v_slot_stride=0), dict(k_page_stride=0), dict(v_page_stride=0)):
        b, keep2 = cache(**bad)
        err(attend(b), text="stride")
        err(append(b), text="stride")
    ones = dict(n_pages=1, page_size=1, n_kv_heads=1, k_page_stride=0, v_page_stride=0, k_slot_stride=0, v_slot_stride=0, k_head_stride=0, v_head_stride=0)
    b, keep2 = cache(**ones)
    assert attend(b, R=0) == 0 and append(b, T=0) == 0


def plan(**change):
    a = dict(lens=P, new=P, table=P, stride=4, width=4, free=P, pool=10, count=P, count_out=P, parents=None, page=16, start=P, slots=P, pos=P, mask=None,
             R=2, T=5, ws=P, nbytes=BIG, stream=None)
    a.update(change)
    return _lib.load().awq_b200_page_plan(*a.values())


def test_page_plan():
    for bad in (dict(R=-1), dict(R=4097), dict(T=-1), dict(T=(1 << 20) + 1), dict(width=-1), dict(pool=-1), dict(page=0), dict(pool=1 << 28),
                dict(width=1 << 28, stride=1 << 28), dict(stride=3), dict(start=None), dict(count=None), dict(count_out=None), dict(lens=None), dict(new=None),
                dict(table=None), dict(free=None), dict(slots=None), dict(pos=None), dict(parents=P), dict(mask=P)):
        err(plan(**bad))
    err(plan(ws=None), _lib.AWQ_ERR_WORKSPACE)


def keep(**change):
    a = dict(kv=P, s0=1 << 20, s1=1 << 18, s2=4096, s3=256, s4=128, layers=2, pages=10, page=16, heads=2, dim=128, table=P, stride=4, width=4, lens=P,
             lens_out=P, start=P, kept=P, path=P, free=P, pool=10, count=P, count_out=P, R=2, T=5, ws=P, nbytes=BIG, stream=None)
    a.update(change)
    return _lib.load().awq_b200_page_keep(*a.values())


def test_page_keep():
    for bad in (dict(R=-1), dict(R=4097), dict(T=-1), dict(layers=-1), dict(layers=5000), dict(pages=0), dict(page=0), dict(heads=0), dict(dim=0), dict(dim=12),
                dict(pages=1 << 28), dict(stride=3), dict(s0=4), dict(s3=-8), dict(count=None), dict(count_out=None), dict(table=None), dict(lens=None),
                dict(lens_out=None), dict(start=None), dict(kept=None), dict(free=None), dict(kv=None), dict(kv=ODD)):
        err(keep(**bad))
    err(keep(nbytes=10), _lib.AWQ_ERR_WORKSPACE)


def lora(**change):
    a = dict(x=P, row=512, A=P, B=P, scales=P, ranks=None, n=3, rank=16, idx=P, base=P, f32=1, res=None, out=P, T=5, K=512, N=256, ws=P, nbytes=BIG,
             stream=None)
    a.update(change)
    return _lib.load().awq_b200_lora_bf16(*a.values())


def test_lora():
    for bad in (dict(T=-1), dict(T=65536), dict(K=0), dict(N=-8), dict(n=-1), dict(rank=0), dict(rank=12), dict(rank=136), dict(K=100), dict(N=12), dict(row=5),
                dict(row=-8), dict(x=None), dict(idx=None), dict(base=None), dict(out=None), dict(A=None), dict(B=None), dict(scales=None), dict(x=ODD),
                dict(A=ODD), dict(B=ODD), dict(base=ODD), dict(res=ODD), dict(out=ODD)):
        err(lora(**bad))
    err(lora(ws=None), _lib.AWQ_ERR_WORKSPACE)
    assert lora(T=0) == 0 and lora(N=0) == 0


def test_lora_refuses_outputs_over_inputs():
    at = lambda n: ctypes.c_void_p(4096 + n)  # noqa: E731
    far, x, out = 1 << 24, 4 * 512 * 2 + 512 * 2, 5 * 256 * 2  # bytes of x and out
    apart = dict(x=at(far), A=at(2 * far), B=at(3 * far), base=at(4 * far), res=at(5 * far), out=at(6 * far))
    for bad in (dict(out=at(far)), dict(out=at(far + x - 16)), dict(out=at(far - out + 16)), dict(out=at(2 * far + 3 * 16 * 512 * 2 - 16)), dict(out=at(3 * far)),
                dict(out=at(4 * far)), dict(out=at(4 * far + 2 * out - 16)), dict(f32=0, out=at(4 * far + 16)), dict(out=at(5 * far + 16))):
        err(lora(**{**apart, **bad}), text="overlap")


def test_handles_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from mlir_air_b200 import ops
    with pytest.raises(_lib.AwqBackendError):
        ops.KVCache(*torch.zeros((2, 3, 16, 2, 64), dtype=torch.bfloat16))
    with pytest.raises(_lib.AwqBackendError):
        ops.LoraAdapters(torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 64, 8, dtype=torch.bfloat16), torch.ones(1))
    with pytest.raises(_lib.AwqBackendError):
        ops.RequestWorkspace(device="cpu")


def test_written_strides_of_zero():
    """Rows, heads or layers that are written must not lie on top of one another: which of them stays would be chance."""
    c, keep2 = cache()
    err(attend(c, orow=0), text="stride")
    err(attend(c, oh=0), text="stride")
    err(append(c, orow=0), text="stride")
    err(append(c, oh=0), text="stride")
    assert attend(c, orow=0, T=0) == 0 and append(c, orow=0, T=0) == 0
    for bad in ("s0", "s1", "s2", "s3", "s4"):
        err(keep(**{bad: 0}), text="stride")
    err(keep(s1=0, layers=1), text="stride")
