"""The paged cache's operators on the CPU: what the entry points refuse before any launch (the
pointers are never dereferenced), and the plain model of the page bookkeeping."""
from __future__ import annotations

import ctypes

import pytest
import torch

import ytensor_amd as yt
from paged_ref import Pages, path_of, select
from ytensor_amd import _lib

FAKE = ctypes.c_void_p(4096)
I3 = _lib.i64array([128, 128, 128])


def attn(lib, sparse=False, **kw):
    a = dict(dtype=_lib.BF16, B=2, Hq=4, Hkv=2, T=3, d=128, Q=FAKE, q=I3, Kn=FAKE, kn=I3, Vn=FAKE, vn=I3, Kp=FAKE,
             Vp=FAKE, p=I3, pages=8, page=16, sums=FAKE, ss=_lib.i64array([128, 128]), table=FAKE, ld=4, columns=4,
             kv_len=FAKE, parents=None, ldp=3, new_len=None, top_k=2, sel=FAKE, O=FAKE, o=I3, ws=FAKE, bytes=1 << 40)
    a.update(kw)
    head = (a["dtype"], a["B"], a["Hq"], a["Hkv"], a["T"], a["d"], a["Q"], a["q"], a["Kn"], a["kn"], a["Vn"], a["vn"],
            a["Kp"], a["Vp"], a["p"], a["pages"], a["page"])
    mid = (a["table"], a["ld"], a["columns"], a["kv_len"], a["parents"], a["ldp"], a["new_len"])
    tail = (a["O"], a["o"], 0.0, a["ws"], a["bytes"], None)
    if sparse:
        return lib.ythip_paged_attn_sparse(*head, a["sums"], a["ss"], *mid, a["top_k"], a["sel"], *tail)
    return lib.ythip_paged_attn(*head, *mid, *tail)


EINVAL, EUNSUP = _lib.YTHIP_EINVAL, _lib.YTHIP_EUNSUPPORTED


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=7), EINVAL, b"dtype"),
    (dict(B=-1), EINVAL, b"negative"),
    (dict(d=96), EUNSUP, b"head dim"),
    (dict(page=48), EINVAL, b"power of two"),
    (dict(page=8), EINVAL, b"power of two"),
    (dict(page=65536), EINVAL, b"power of two"),
    (dict(Hq=5), EINVAL, b"heads"),
    (dict(Hkv=0), EINVAL, b"heads"),
    (dict(columns=70000, ld=70000), EUNSUP, b"columns"),
    (dict(columns=65536, ld=65536, page=32768), EUNSUP, b"2^30"),
    (dict(columns=65536, ld=65536, page=16384, B=17), EUNSUP, b"2^34"),
    (dict(parents=FAKE, T=4097, ldp=4097), EUNSUP, b"tree"),
    (dict(T=1 << 29), EUNSUP, b"new tokens"),
    (dict(kn=_lib.i64array([128, 128, 1 << 24])), EUNSUP, b"stride"),
    (dict(p=_lib.i64array([128, 128, -128])), EUNSUP, b"stride"),
    (dict(B=65536), EUNSUP, b"65535"),
    (dict(parents=FAKE, ldp=2), EINVAL, b"parents"),
    (dict(Q=None), EINVAL, b"NULL"),
    (dict(O=None), EINVAL, b"NULL"),
    (dict(kv_len=None), EINVAL, b"NULL"),
    (dict(Vn=None), EINVAL, b"together"),
    (dict(kn=None), EINVAL, b"together"),
    (dict(table=None), EINVAL, b"NULL"),
    (dict(Kp=None), EINVAL, b"NULL"),
    (dict(ld=3), EINVAL, b"stride"),
    (dict(Q=ctypes.c_void_p(4098)), EUNSUP, b"aligned"),
    (dict(Vp=ctypes.c_void_p(4104)), EUNSUP, b"aligned"),
    (dict(p=_lib.i64array([128, 100, 128])), EUNSUP, b"aligned"),
])
def test_attention_refuses(sparse, change, status, text):
    lib = yt.load()
    assert attn(lib, sparse, **change) == status
    assert text in lib.ythip_last_error()


@pytest.mark.parametrize("change,status,text", [
    (dict(top_k=0), EINVAL, b"top_k"), (dict(top_k=4097), EINVAL, b"top_k"), (dict(sel=None), EINVAL, b"sel"),
    (dict(sums=None), EINVAL, b"sums"), (dict(bytes=16), EINVAL, b"workspace"), (dict(ws=None), EINVAL, b"workspace"),
    (dict(ws=ctypes.c_void_p(4100)), EINVAL, b"aligned"),
])
def test_sparse_attention_refuses(change, status, text):
    lib = yt.load()
    assert attn(lib, True, **change) == status
    assert text in lib.ythip_last_error()


def test_nothing_to_do_launches_nothing():
    lib = yt.load()
    for change in (dict(B=0), dict(T=0), dict(Hq=0)):
        assert attn(lib, **change) == 0 and attn(lib, True, **change) == 0


def pool(n=1, **kw):
    a = dict(data=4096, layer_stride=1 << 20, page_stride=1 << 12, page_bytes=1 << 12)
    a.update(kw)
    return (_lib.PagePool * n)(*[_lib.PagePool(a["data"], a["layer_stride"], a["page_stride"], a["page_bytes"])] * n)


def test_bookkeeping_refuses():
    lib = yt.load()
    st = lambda **k: [{**dict(B=2, c=4, P=8, page=16, ref=FAKE, t=FAKE, ld=4, len=FAKE, ro=FAKE, to=FAKE, ldo=4, lo=FAKE), **k}[x] for x in ("B", "c", "P", "page", "ref", "t", "ld", "len", "ro", "to", "ldo", "lo")]  # noqa: E731

    def grow(n=FAKE, **k):
        s = st(**k)
        return lib.ythip_cache_grow(*s[:8], n, *s[8:], None, None)

    def fork(n=2, src=FAKE, np=1, layers=1, pools=None, ws=FAKE, nb=1 << 20, **k):
        s = st(**k)
        return lib.ythip_cache_fork(*s[:8], n, src, FAKE, *s[8:], np, layers, pools or pool(), None, ws, nb, None)

    def free(n=2, seqs=FAKE, **k):
        s = st(**k)
        return lib.ythip_cache_free(*s[:8], n, seqs, *s[8:], None, None)

    def compact(live=FAKE, np=1, pools=None, ws=FAKE, nb=1 << 20, **k):
        s = st(**k)
        return lib.ythip_cache_compact(*s[:8], *s[8:11], live, np, 1, pools or pool(), ws, nb, None)

    for call in (grow, fork, free, compact):
        assert call(B=-1) == EINVAL
        assert call(page=24) == EINVAL and b"power of two" in lib.ythip_last_error()
        assert call(ref=None) == EINVAL and call(ro=None) == EINVAL
        assert call(t=None) == EINVAL and call(len=None) == EINVAL and call(to=None) == EINVAL
        assert call(ld=3) == EINVAL and call(ldo=3) == EINVAL
        assert call(ldo=5) == EINVAL and b"two strides" in lib.ythip_last_error()
        assert call(c=65537, ld=65537, ldo=65537) == EUNSUP
    assert grow(n=None) == EINVAL and grow(B=4097) == EUNSUP
    assert fork(n=-1) == EINVAL and fork(src=None) == EINVAL and fork(n=4097) == EUNSUP
    assert fork(nb=16) == EINVAL and fork(ws=None) == EINVAL and fork(ws=ctypes.c_void_p(4100)) == EINVAL
    assert free(n=-1) == EINVAL and free(seqs=None) == EINVAL
    assert compact(live=None) == EINVAL and compact(nb=16) == EINVAL and compact(ws=None) == EINVAL
    for call in (fork, compact):
        assert call(np=5, pools=pool(5)) == EINVAL and call(np=-1) == EINVAL
        for bad in (dict(data=0), dict(data=4098), dict(page_bytes=0), dict(page_bytes=10), dict(page_stride=6)):
            assert call(pools=pool(**bad)) == EINVAL and b"pool 0" in lib.ythip_last_error()
    assert lib.ythip_cache_copy_pages(-1, 1, FAKE, FAKE, 1, 1, pool(), None, None) == EINVAL
    assert lib.ythip_cache_copy_pages(8, 1, None, FAKE, 1, 1, pool(), None, None) == EINVAL
    assert lib.ythip_cache_copy_pages(8, 1, FAKE, FAKE, 1, -1, pool(), None, None) == EINVAL
    assert lib.ythip_cache_copy_pages(8, 0, None, None, 1, 1, pool(), None, None) == 0


@pytest.mark.parametrize("change,status", [
    (dict(dtype=9), EINVAL), (dict(L=-1), EINVAL), (dict(d=0), EINVAL), (dict(d=12), EUNSUP), (dict(d=4096), EUNSUP),
    (dict(page=17), EINVAL), (dict(Kn=None), EINVAL), (dict(Kp=None), EINVAL), (dict(ss=None), EINVAL),
    (dict(table=None), EINVAL), (dict(kv_len=None), EINVAL), (dict(ld=1), EINVAL),
    (dict(Vp=ctypes.c_void_p(4100)), EUNSUP), (dict(ns=_lib.i64array([128, 128, 4, 128])), EUNSUP),
    (dict(L=1 << 20, B=1 << 10, Hkv=8), EUNSUP), (dict(B=0), 0), (dict(T=0), 0),
])
def test_append_refuses(change, status):
    lib = yt.load()
    i4 = _lib.i64array([128] * 4)
    a = dict(dtype=_lib.F16, L=2, B=2, Hkv=2, T=3, d=128, Kn=FAKE, Vn=FAKE, ns=i4, Kp=FAKE, Vp=FAKE, ps=i4, pages=8,
             page=16, sums=FAKE, ss=_lib.i64array([1, 1, 1]), table=FAKE, ld=4, columns=4, kv_len=FAKE)
    a.update(change)
    assert lib.ythip_cache_append(*a.values(), None, None, 3, None) == status


def test_python_layer_refuses_host_tensors():
    q, pool4 = torch.zeros(1, 2, 1, 64), torch.zeros(4, 1, 16, 64)
    table, one = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        yt.paged_attention(q, None, None, pool4, pool4, table, one)
    with pytest.raises(ValueError, match="at least one page"):
        yt.paged_sparse_attention(q, None, None, pool4, pool4, pool4[:, :, 0], table, one, 0)
    with pytest.raises(ValueError, match="device"):
        yt.cache_grow(one, table, one, one, 16)
    with pytest.raises(ValueError, match="device"):
        yt.cache_copy_pages([pool4[None]], one, one)


def test_model_of_the_pages():
    """The plain model itself, on a case worked out by hand."""
    m = Pages(torch.tensor([1, 0, 1, 0, 0]), torch.tensor([[2, 0, -1], [-1, -1, -1], [-1, -1, -1]]),
              torch.tensor([20, 0, 0]), 16, [torch.arange(5.0)[None, :, None]])
    m.fork([0, 0, 0], [1, 1, 0])                     # one, a second mention, an occupied one
    assert m.ref == [1, 1, 2, 0, 0] and m.table[1] == [2, 1, -1] and m.len == [20, 20, 0] and m.status == 2
    assert m.pools[0][0, 1, 0] == 0
    m.grow([13, 0, 17])                              # one page, none, two: one too few
    assert m.table[0] == [2, 0, 3] and m.len == [33, 20, 0] and m.status == 6
    m.free([0, 0, 7])
    assert m.ref == [0, 1, 1, 0, 0] and m.table[0] == [-1, -1, -1] and m.status == 7
    assert m.compact() == 2 and m.ref == [1, 1, 0, 0, 0] and m.table[1] == [0, 1, -1]
    assert path_of([-1, 0, 0, 2, 9], 3) == [0, 2, 3] and path_of([-1, 0, 0, 2, 9], 4) == [4]
    sums = torch.tensor([[[1.0] * 64], [[3.0] * 64], [[3.0] * 64], [[0.0] * 64]])
    s = select(torch.ones(1, 1, 1, 64), sums, torch.tensor([[0, 1, 2, 3]]), torch.tensor([50]), 16, 2)
    assert s.tolist() == [[[[1, 3]]]]


def test_attention_workspace():
    """None where a sequence stays with one workgroup; else room for every partial, whatever the lengths."""
    lib = yt.load()
    size = lambda B, T, columns, page=64, G=2, d=128: int(lib.ythip_paged_attn_workspace_size(_lib.BF16, B, 8 * G, 8, T, d, columns, page))  # noqa: E731
    assert size(1, 1, 5) == 0 and size(64, 1, 5) == 0 and size(1, 1, 0) == 0 and size(0, 1, 5) == 0
    big = size(1, 1, 2048)
    assert big > 0 and big % (8 * 2 * 130 * 4) == 0
    st = attn(lib, Hq=16, Hkv=8, T=1, B=1, columns=2048, ld=2048, page=64, bytes=big - 1)
    assert st == EINVAL and b"workspace of" in lib.ythip_last_error()
    assert attn(lib, Hq=16, Hkv=8, T=1, B=1, columns=2048, ld=2048, page=64, ws=None) == EINVAL
    sparse = int(lib.ythip_paged_attn_sparse_workspace_size(_lib.BF16, 2, 16, 8, 3, 128, 100, 64, 4))
    assert sparse >= 2 * 8 * 3 * 100 * 8
