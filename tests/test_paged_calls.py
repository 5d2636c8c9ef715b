"""What the paged cache's entry points refuse before any launch, on the CPU (the pointers are never dereferenced)."""
from __future__ import annotations

import ctypes

import pytest
import torch

import ytensor_amd as yt
from ytensor_amd import _lib, paged

FAKE, OTHER = ctypes.c_void_p(4096), ctypes.c_void_p(8192)
EINVAL, EUNSUP = _lib.YTHIP_EINVAL, _lib.YTHIP_EUNSUPPORTED


def append(lib, to, **kw):
    i4 = _lib.i64array([128] * 4)
    a = dict(dtype=_lib.BF16, L=2, B=2, Hkv=2, T=3, d=128, Kn=FAKE, Vn=FAKE, ns=i4, Kp=FAKE, Vp=FAKE, ps=i4, pages=8,
             page=16, sums=FAKE, ss=_lib.i64array([1, 1, 1]), table=FAKE, ld=4, columns=4, kv_len=FAKE, count=OTHER,
             path=None, ldp=3)
    a.update(kw)
    return (lib.ythip_cache_append_to(*a.values(), None, None) if to else lib.ythip_cache_append(*a.values(), None))


@pytest.mark.parametrize("change,status,text", [
    (dict(count=None), EINVAL, b"new_len"), (dict(dtype=9), EINVAL, b"dtype"), (dict(d=12), EUNSUP, b"rows of"),
    (dict(page=17), EINVAL, b"power of two"), (dict(Kn=None), EINVAL, b"NULL"), (dict(ss=None), EINVAL, b"NULL"),
    (dict(kv_len=None), EINVAL, b"NULL"), (dict(ld=1), EINVAL, b"stride"), (dict(Vp=ctypes.c_void_p(4100)), EUNSUP, b"aligned"),
])
def test_append_to_given_lengths_refuses(change, status, text):
    lib = yt.load()
    assert append(lib, True, **change) == status
    assert b"ythip_cache_append_to" in lib.ythip_last_error() and text in lib.ythip_last_error()


def test_dims_of_one_element_have_no_stride():
    """A view whose only odd strides are those of dims of one element is taken as it is; others are copied, to
    strides of their own."""
    odd = torch.empty_strided((1, 2, 1, 64), (1001, 64, 7, 1), dtype=torch.bfloat16)
    t, at, st = paged._rows(odd, 2)
    assert t is odd and at == odd.data_ptr() and st == (1001, 64, 7, 1) and paged._real(odd) == (0, 64, 0, 1)
    for stride in ((72, 65, 7, 1), (128, 1, 1, 2)):
        t, at, st = paged._rows(torch.empty_strided((1, 2, 1, 64), stride, dtype=torch.bfloat16), 2)
        assert st == (128, 64, 64, 1) and at == t.data_ptr() and at % 16 == 0
    assert paged._pool_layout((1, 1, 3, 16), (7, 5, 16, 1), 2) == (1, 1, 0, 0, 96)
    assert paged._pool_layout((2, 4, 3, 16), (200, 50, 16, 1), 2) == (2, 4, 400, 100, 96)


def test_strides_that_matter_are_still_refused():
    lib, odd = yt.load(), _lib.i64array([100, 128, 128, 128])
    assert append(lib, False, ns=odd) == EUNSUP and append(lib, False, ps=odd) == EUNSUP
    assert b"aligned" in lib.ythip_last_error()
    for axis in range(4):
        ns = _lib.i64array([100 if i == axis else 128 for i in range(4)])
        assert append(lib, False, ns=ns) == EUNSUP


@pytest.mark.parametrize("empty", ["L", "B", "Hkv", "T", "pages", "columns"])
def test_appends_of_nothing_take_no_pointers(empty):
    """An empty tensor has no address."""
    lib = yt.load()
    none = dict(Kn=None, Vn=None, Kp=None, Vp=None, sums=None, table=None) if empty != "columns" else dict(table=None)
    if empty not in ("B", "columns"):
        del none["table"]
    for to in (False, True):
        assert append(lib, to, **{empty: 0, **none}) == 0


def test_bookkeeping_without_columns_takes_no_table():
    lib = yt.load()
    # (not 0 here, where asking for the last launch's error finds no GPU)
    assert lib.ythip_cache_free(2, 0, 8, 16, FAKE, None, 0, FAKE, 0, None, FAKE, None, 0, FAKE, None, None) != EINVAL
    assert lib.ythip_cache_free(2, 1, 8, 16, FAKE, None, 1, FAKE, 0, None, FAKE, None, 1, FAKE, None, None) == EINVAL


def test_more_workgroups_than_a_launch_holds():
    """A grid's dimension has fewer than 2^32 threads: refused before anything runs."""
    lib = yt.load()
    for change in (dict(L=1 << 10, B=1 << 10, Hkv=64), dict(L=1 << 8, B=1 << 8, Hkv=256, page=512),
                   dict(L=1 << 7, B=1 << 7, Hkv=256, page=1024)):
        for to in (False, True):
            assert append(lib, to, **change) == EUNSUP and b"pages to write" in lib.ythip_last_error()
    i3 = _lib.i64array([128] * 3)

    def attention(B, Hq, Hkv, T, columns):
        return lib.ythip_paged_attn(_lib.BF16, B, Hq, Hkv, T, 128, FAKE, i3, FAKE, i3, FAKE, i3, FAKE, FAKE, i3, 8, 16, FAKE,
                                    columns, columns, FAKE, None, 0, None, FAKE, i3, 0.0, FAKE, 1 << 62, None)

    assert attention(65535, 512, 512, 1, 4) == EUNSUP and b"workgroups" in lib.ythip_last_error()
    assert attention(2, 256, 1, 1 << 21, 64) == EUNSUP and b"workgroups" in lib.ythip_last_error()


@pytest.mark.parametrize("to", [False, True])
@pytest.mark.parametrize("stride", [2, 0, -3])
def test_append_refuses_paths_that_overlap(to, stride):
    lib = yt.load()
    assert append(lib, to, path=FAKE, ldp=stride) == EINVAL and b"path" in lib.ythip_last_error()


def test_sparse_workspace_parts_are_aligned():
    """The ranks lie in front of the partials, which are read 16 bytes at a time."""
    lib = yt.load()
    size = lambda B, Hkv, T, columns: int(lib.ythip_paged_attn_sparse_workspace_size(_lib.BF16, B, 2 * Hkv, Hkv, T, 64, columns, 16, 5))  # noqa: E731
    for B, Hkv, T, columns in ((1, 1, 1, 1251), (1, 1, 1, 129), (3, 1, 5, 1001), (1, 7, 1, 131)):
        assert B * Hkv * T * columns % 2 == 1 and size(B, Hkv, T, columns) % 16 == 0
        assert size(B, Hkv, T, columns) >= 8 * B * Hkv * T * columns


def test_one_range_takes_no_workspace():
    """Where the row tiles alone fill the GPU no sequence is cut, and there are no partials to hold."""
    lib = yt.load()
    size = lambda B, Hkv, T, columns: int(lib.ythip_paged_attn_workspace_size(_lib.BF16, B, 2 * Hkv, Hkv, T, 128, columns, 64))  # noqa: E731
    assert size(1, 8, 4096, 64) == 0 and size(3, 8, 4096, 2048) == 0 and size(2, 8, 2100, 300) == 0
    assert size(1, 8, 1024, 64) > 0 and size(16, 8, 2048, 100) > 0


def test_append_refuses_one_array_of_lengths():
    """A grow in place and an append that is given its lengths as both: no row would be written."""
    lib = yt.load()
    assert append(lib, True, kv_len=FAKE, count=FAKE) == EINVAL and b"one array" in lib.ythip_last_error()


def test_sparse_attention_refuses_more_tokens_than_its_grid_holds():
    lib, i3 = yt.load(), _lib.i64array([128] * 3)

    def sparse(Hkv, T):
        return lib.ythip_paged_attn_sparse(_lib.BF16, 1, Hkv, Hkv, T, 128, FAKE, i3, None, None, None, None, FAKE, FAKE, i3, 8, 16,
                                           FAKE, i3, FAKE, 4, 4, FAKE, None, 0, None, 2, FAKE, FAKE, i3, 0.0, FAKE, 0, None)

    assert sparse(8, 8192) == EUNSUP and b"65535" in lib.ythip_last_error()
    assert sparse(5, 13107) == EINVAL and b"workspace" in lib.ythip_last_error()  # 65535: taken, and stopped further on


def test_grow_refuses_its_counts_as_the_lengths_to_write():
    lib = yt.load()
    grow = lambda n, out: lib.ythip_cache_grow(2, 4, 8, 16, FAKE, FAKE, 4, FAKE, n, FAKE, FAKE, 4, out, None, None)  # noqa: E731
    assert grow(OTHER, OTHER) == EINVAL and b"one array" in lib.ythip_last_error()
    assert grow(None, OTHER) == EINVAL and b"NULL" in lib.ythip_last_error()
