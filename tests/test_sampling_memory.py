"""What token_probs and verify_drafts write must not lie over what they read, on the CPU: refused before any launch (the
pointers are never dereferenced)."""
from __future__ import annotations

import ctypes

import pytest

import ytensor_amd as yt
from ytensor_amd import _lib

EINVAL, B, T = _lib.YTHIP_EINVAL, 3, 8
# a region of 64 KB for each argument
AT = {name: (i + 1) << 16 for i, name in enumerate(("target", "tokens", "parents", "tree_len", "u", "u_next", "path", "kept", "next", "ws"))}


def verify(ld=(T, T, T, T), **at):
    p = {name: ctypes.c_void_p(at.get(name, x)) for name, x in AT.items()}
    i2 = _lib.i64array([T * 50, 50])
    return yt.load().ythip_verify_drafts(_lib.F32, B, T, 50, p["target"], i2, None, i2, p["tokens"], ld[0], p["parents"], ld[1], p["tree_len"], p["u"],
                                         ld[2], p["u_next"], p["path"], ld[3], p["kept"], p["next"], p["ws"], 1 << 15, None)


@pytest.mark.parametrize("at", [
    dict(kept=AT["tree_len"]), dict(kept=AT["tree_len"] + 4 * (B - 1)), dict(path=AT["tokens"]), dict(path=AT["tokens"] + 4 * (B * T - 1)),
    dict(path=AT["parents"]), dict(path=AT["u"]), dict(kept=AT["u_next"] - 4), dict(next=AT["tree_len"] + 4), dict(next=AT["tokens"]),
    dict(path=AT["tree_len"] - 4 * B * T + 4), dict(next=AT["ws"]), dict(path=AT["ws"] + 8),
])
def test_outputs_over_inputs(at):
    assert verify(**at) == EINVAL
    assert b"over what is read" in yt.load().ythip_last_error()


@pytest.mark.parametrize("at", [dict(kept=AT["next"]), dict(kept=AT["next"] + 4), dict(path=AT["kept"]), dict(next=AT["path"] + 4 * (B * T - 1))])
def test_outputs_over_each_other(at):
    assert verify(**at) == EINVAL
    assert b"over each other" in yt.load().ythip_last_error()


def test_rows_in_each_other_s_gaps():
    """Rows of tokens and of the path that alternate, an element too near or too far."""
    wide = (2 * T, T, T, 2 * T)
    for by in (T - 1, T + 1, 3 * T - 1, -T + 1):
        assert verify(ld=wide, path=AT["tokens"] + 4 * by) == EINVAL
        assert b"over what is read" in yt.load().ythip_last_error()
    # a row of counts that reaches out of a gap
    assert verify(ld=(T + B, T, T, T), kept=AT["tokens"] + 4 * (T + 1)) == EINVAL


def probs(at, rows=3, n=100, ld=100, ldo=100, dtype=_lib.F32):
    return yt.load().ythip_token_probs(dtype, rows, n, ctypes.c_void_p(1 << 20), ld, 1.0, ctypes.c_void_p((1 << 20) + at), ldo, None, 0, None)


@pytest.mark.parametrize("kw", [
    dict(at=4), dict(at=-4), dict(at=400), dict(at=-800), dict(at=0, ldo=101), dict(at=0, dtype=_lib.BF16), dict(at=0, dtype=_lib.F16, ld=200),
    dict(at=4 * 99, ld=200, ldo=200), dict(at=4 * 101, ld=200, ldo=200), dict(at=396, rows=1), dict(at=500, ld=150, ldo=160),
])
def test_probs_over_logits(kw):
    assert probs(**kw) == EINVAL
    assert b"over logits" in yt.load().ythip_last_error()
