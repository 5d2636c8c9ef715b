"""4-bit pages on the CPU: what the entry points refuse before any launch (the pointers are never dereferenced), and the
plain model against itself."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import q4_ref
import ytensor_amd as yt
from ytensor_amd import _lib

FAKE, OTHER = ctypes.c_void_p(4096), ctypes.c_void_p(8192)
EINVAL, EUNSUP = _lib.YTHIP_EINVAL, _lib.YTHIP_EUNSUPPORTED
I2, I3, I4 = (_lib.i64array([128] * n) for n in (2, 3, 4))


def append(lib, **kw):
    a = dict(dtype=_lib.BF16, L=2, B=2, Hkv=2, T=3, d=128, Kn=FAKE, Vn=FAKE, ns=I4, Kp=FAKE, Vp=FAKE, ps=I3, pages=8, page=16,
             table=FAKE, ld=4, columns=4, kv_len=FAKE, n_new=None, new_len=OTHER, path=None, ldp=3)
    a.update(kw)
    return lib.ythip_cache_append_q4(*a.values(), None, None)


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=9), EINVAL, b"dtype"), (dict(L=-1), EINVAL, b"negative"), (dict(T=-1), EINVAL, b"negative"),
    (dict(d=96), EUNSUP, b"head dim"), (dict(page=8), EINVAL, b"power of two"), (dict(page=65536), EINVAL, b"power of two"),
    (dict(n_new=FAKE), EINVAL, b"both"), (dict(new_len=FAKE), EINVAL, b"one array"), (dict(columns=70000, ld=70000), EUNSUP, b"columns"),
    (dict(columns=65536, ld=65536, page=32768), EUNSUP, b"2^30"), (dict(Kn=None), EINVAL, b"NULL"), (dict(Vp=None), EINVAL, b"NULL"),
    (dict(ns=None), EINVAL, b"NULL"), (dict(ps=None), EINVAL, b"NULL"), (dict(table=None), EINVAL, b"NULL"), (dict(kv_len=None), EINVAL, b"NULL"),
    (dict(ld=3), EINVAL, b"stride"), (dict(path=FAKE, ldp=2), EINVAL, b"path"), (dict(Kp=ctypes.c_void_p(4104)), EUNSUP, b"aligned"),
    (dict(Vn=ctypes.c_void_p(4104)), EUNSUP, b"aligned"), (dict(ps=_lib.i64array([128, 100, 128])), EUNSUP, b"aligned"),
    (dict(ns=_lib.i64array([128, 128, 4, 128])), EUNSUP, b"aligned"), (dict(L=1 << 12, B=1 << 12, Hkv=1 << 4), EUNSUP, b"workgroups"),
])
def test_append_refuses(change, status, text):
    lib = yt.load()
    assert append(lib, **change) == status
    assert text in lib.ythip_last_error()


@pytest.mark.parametrize("empty", ["L", "B", "Hkv", "T", "pages", "columns"])
def test_appends_of_nothing(empty):
    assert append(yt.load(), Kn=None, Vn=None, Kp=FAKE, **{empty: 0}) == 0


def unpack(lib, **kw):
    a = dict(dtype=_lib.F32, L=2, pages=3, Hkv=2, page=16, d=64, Kp=FAKE, Vp=FAKE, ps=I3, K=FAKE, V=FAKE)
    a.update(kw)
    return lib.ythip_cache_unpack_q4(*a.values(), None)


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=3), EINVAL, b"dtype"), (dict(pages=-1), EINVAL, b"negative"), (dict(d=32), EUNSUP, b"head dim"), (dict(page=24), EINVAL, b"power of two"),
    (dict(Kp=None), EINVAL, b"NULL"), (dict(ps=None), EINVAL, b"NULL"), (dict(K=None), EINVAL, b"NULL"), (dict(V=ctypes.c_void_p(4100)), EUNSUP, b"aligned"),
    (dict(Kp=ctypes.c_void_p(4100)), EUNSUP, b"aligned"), (dict(ps=_lib.i64array([16, 8, 16])), EUNSUP, b"aligned"),
    (dict(pages=1 << 20, Hkv=1 << 10), EUNSUP, b"workgroups"),
])
def test_unpack_refuses(change, status, text):
    lib = yt.load()
    assert unpack(lib, **change) == status
    assert text in lib.ythip_last_error()
    assert unpack(lib, L=0, Kp=None, ps=None) == 0


def attn(lib, **kw):
    a = dict(dtype=_lib.BF16, B=2, Hq=4, Hkv=2, T=3, d=128, Q=FAKE, q=I3, Kn=FAKE, kn=I3, Vn=FAKE, vn=I3, Kp=FAKE, Vp=FAKE, p=I2,
             pages=8, page=16, table=FAKE, ld=4, columns=4, kv_len=FAKE, parents=None, ldp=3, new_len=None, window=0, sinks=0,
             O=FAKE, o=I3, scale=0.0, ws=FAKE, bytes=1 << 40)
    a.update(kw)
    return lib.ythip_paged_attn_q4(*a.values(), None)


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=7), EINVAL, b"dtype"), (dict(B=-1), EINVAL, b"negative"), (dict(d=96), EUNSUP, b"head dim"), (dict(page=48), EINVAL, b"power of two"),
    (dict(Hq=5), EINVAL, b"heads"), (dict(Hkv=0), EINVAL, b"heads"), (dict(window=-1), EINVAL, b"window"), (dict(sinks=-1), EINVAL, b"sinks"),
    (dict(columns=70000, ld=70000), EUNSUP, b"columns"), (dict(columns=65536, ld=65536, page=16384, B=17), EUNSUP, b"2^34"),
    (dict(parents=FAKE, T=4097, ldp=4097), EUNSUP, b"tree"), (dict(T=1 << 29), EUNSUP, b"new tokens"), (dict(B=65536), EUNSUP, b"65535"),
    (dict(Q=None), EINVAL, b"NULL"), (dict(p=None), EINVAL, b"NULL"), (dict(kv_len=None), EINVAL, b"NULL"), (dict(Vn=None), EINVAL, b"together"),
    (dict(table=None), EINVAL, b"NULL"), (dict(Kp=None), EINVAL, b"NULL"), (dict(ld=3), EINVAL, b"stride"), (dict(parents=FAKE, ldp=2), EINVAL, b"parents"),
    (dict(Q=ctypes.c_void_p(4098)), EUNSUP, b"aligned"), (dict(Vp=ctypes.c_void_p(4104)), EUNSUP, b"aligned"), (dict(p=_lib.i64array([136, 128])), EUNSUP, b"aligned"),
    (dict(columns=4096, ld=4096, ws=None), EINVAL, b"workspace"), (dict(columns=4096, ld=4096, bytes=64), EINVAL, b"workspace"),
    (dict(columns=4096, ld=4096, ws=ctypes.c_void_p(4104)), EINVAL, b"aligned"),
])
def test_attention_refuses(change, status, text):
    lib = yt.load()
    assert attn(lib, **change) == status
    assert text in lib.ythip_last_error()
    assert b"ythip_paged_attn_q4" in lib.ythip_last_error()


@pytest.mark.parametrize("change,status,text", [(dict(window=-3), EINVAL, b"window"), (dict(sinks=-3), EINVAL, b"sinks"), (dict(d=80), EUNSUP, b"head dim"),
                                                (dict(ws=None, columns=4096, ld=4096, window=9000), EINVAL, b"workspace")])
def test_window_refuses(change, status, text):
    lib = yt.load()
    a = dict(dtype=_lib.BF16, B=2, Hq=4, Hkv=2, T=3, d=128, Q=FAKE, q=I3, Kn=FAKE, kn=I3, Vn=FAKE, vn=I3, Kp=FAKE, Vp=FAKE, p=I3,
             pages=8, page=16, table=FAKE, ld=4, columns=4, kv_len=FAKE, parents=None, ldp=3, new_len=None, window=5, sinks=1,
             O=FAKE, o=I3, scale=0.0, ws=FAKE, bytes=1 << 40)
    a.update(change)
    assert lib.ythip_paged_attn_window(*a.values(), None) == status
    assert text in lib.ythip_last_error() and b"ythip_paged_attn_window" in lib.ythip_last_error()


def test_a_window_of_all_rows_needs_what_no_window_does():
    lib = yt.load()
    args = (_lib.BF16, 2, 8, 4, 3, 128, 100, 32)
    plain = lib.ythip_paged_attn_workspace_size(*args)
    assert lib.ythip_paged_attn_window_workspace_size(*args, 100 * 32 + 3, 9) == plain == lib.ythip_paged_attn_window_workspace_size(*args, 0, 9)
    assert 0 < lib.ythip_paged_attn_window_workspace_size(*args, 1000, 4) <= plain
    q4 = lib.ythip_paged_attn_q4_workspace_size
    assert q4(*args, 1 << 30, 0) == q4(*args, 0, 0) > 0 == q4(*args, -1, 0)


def test_sizes():
    for page in (16, 64, 32768):
        assert yt.cache_q4_bytes(page, 128) == page * 68 and yt.cache_q4_bytes(page, 64) == page * 34
    for page, d in ((8, 128), (24, 64), (16, 96), (0, 64)):
        with pytest.raises(ValueError):
            yt.cache_q4_bytes(page, d)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("d", [64, 128])
def test_the_model_of_blocks(dtype, which, d):
    """Whole tensors and row by row give the same bytes, and values no further off than half a step."""
    g = torch.Generator().manual_seed(d)
    x = torch.randn(16, d, generator=g) * torch.exp2(torch.randint(-9, 9, (16, 1), generator=g).float())
    x[3], x[4, :32] = 0.0, 7.0
    x = x.to(dtype)
    codes, scales = q4_ref.rows(x)
    block = torch.zeros(16 * (d // 2 + d // 32), dtype=torch.uint8)
    for r in range(16):
        q4_ref.put(block, r, codes[r], scales[r], 16, d, which)
    assert torch.equal(block, q4_ref.pack(x, which))
    v = q4_ref.values(block, 16, d, which)
    unit = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    step = torch.where(v.abs() >= 4 * unit, 2.0, torch.where(v.abs() >= 2 * unit, 1.0, 0.5)) * unit
    assert ((v - x.double()).abs() <= step / 2 + (v.abs() >= 6 * unit) * 0.0).all()


def test_the_model_of_a_group():
    """Ties, the borders of a scale and the ends of its range."""
    def of(values, dtype=torch.float32):
        return q4_ref.group([float(v) for v in values] + [0.0] * (32 - len(values)), dtype)
    codes, byte = of([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0])
    assert byte == 127 and codes[:10] == [7, 0, 2, 2, 4, 4, 6, 6, 8, 14]
    assert of([7.0])[1] == 127 and of([math.nextafter(7.0, 8.0)])[1] == 128 and of([3.5])[1] == 126 and of([0.0])[1] == 2
    assert of([2.0 ** -140])[1] == 2 and of([3e38])[1] == 252 and of([65504.0], torch.float16) == ([7] + [0] * 31, 140)
    assert of([math.nan])[1] == 255 == of([1.0, -math.inf])[1]
