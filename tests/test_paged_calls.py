"""What the paged cache's entry points refuse before any launch, on the CPU (the pointers are never dereferenced)."""
from __future__ import annotations

import ctypes

import pytest

import ytensor_amd as yt
from ytensor_amd import _lib

FAKE = ctypes.c_void_p(4096)
EINVAL, EUNSUP = _lib.YTHIP_EINVAL, _lib.YTHIP_EUNSUPPORTED


def append(lib, to, **kw):
    i4 = _lib.i64array([128] * 4)
    a = dict(dtype=_lib.BF16, L=2, B=2, Hkv=2, T=3, d=128, Kn=FAKE, Vn=FAKE, ns=i4, Kp=FAKE, Vp=FAKE, ps=i4, pages=8,
             page=16, sums=FAKE, ss=_lib.i64array([1, 1, 1]), table=FAKE, ld=4, columns=4, kv_len=FAKE, count=FAKE,
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
