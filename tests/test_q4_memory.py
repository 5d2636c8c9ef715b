"""Where the values of 4-bit pages are written, on the CPU: never over the pools or each other (refused before any launch;
the pointers are never dereferenced)."""
from __future__ import annotations

import ctypes

import pytest

import ytensor_amd as yt
from ytensor_amd import _lib

L, P, H, PAGE, D = 2, 3, 2, 16, 64
BLOCK, VALUES = PAGE * 34, L * P * H * PAGE * D * 4
AT = {name: (i + 1) << 20 for i, name in enumerate(("Kp", "Vp", "K", "V"))}


@pytest.mark.parametrize("at,text", [
    (dict(V=AT["K"]), b"over each other"), (dict(V=AT["K"] + VALUES - 16), b"over each other"), (dict(K=AT["V"] - VALUES + 16), b"over each other"),
    (dict(K=AT["Kp"]), b"over the pools"), (dict(K=AT["Vp"] + L * P * H * BLOCK - 16), b"over the pools"), (dict(V=AT["Kp"] - VALUES + 16), b"over the pools"),
])
def test_values_over_other_memory(at, text):
    p = {name: ctypes.c_void_p(at.get(name, x)) for name, x in AT.items()}
    st = yt.load().ythip_cache_unpack_q4(_lib.F32, L, P, H, PAGE, D, p["Kp"], p["Vp"], _lib.i64array([P * H * BLOCK, H * BLOCK, BLOCK]), p["K"], p["V"], None)
    assert st == _lib.YTHIP_EINVAL
    assert text in yt.load().ythip_last_error()
