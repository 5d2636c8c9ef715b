"""Probabilities and the verification of drafted tokens on the CPU: what the entry points refuse before any launch (the
pointers are never dereferenced), and the plain model."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import ytensor_amd as yt
from sampling_ref import verify as model
from ytensor_amd import _lib

FAKE = ctypes.c_void_p(4096)
EINVAL, EUNSUP = _lib.YTHIP_EINVAL, _lib.YTHIP_EUNSUPPORTED


def probs(lib, **kw):
    a = dict(dtype=_lib.BF16, rows=3, n=100000, x=FAKE, ld=100000, temperature=1.0, p=FAKE, ldo=100000, ws=FAKE, bytes=1 << 30)
    a.update(kw)
    return lib.ythip_token_probs(*a.values(), None)


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=5), EINVAL, b"dtype"), (dict(rows=-1), EINVAL, b"negative"), (dict(n=-1), EINVAL, b"negative"),
    (dict(temperature=0.0), EINVAL, b"temperature"), (dict(temperature=-1.0), EINVAL, b"temperature"),
    (dict(temperature=math.nan), EINVAL, b"temperature"), (dict(temperature=math.inf), EINVAL, b"temperature"),
    (dict(temperature=1e-39), EUNSUP, b"temperature"), (dict(x=None), EINVAL, b"NULL"), (dict(p=None), EINVAL, b"NULL"),
    (dict(ld=99999), EINVAL, b"strides"), (dict(ldo=99999), EINVAL, b"strides"),
    (dict(x=ctypes.c_void_p(4097)), EINVAL, b"within"), (dict(p=ctypes.c_void_p(4098)), EINVAL, b"within"),
    (dict(rows=1 << 22, n=8, ld=8, ldo=8), EUNSUP, b"rows"), (dict(n=(1 << 30) + 1, ld=1 << 31, ldo=1 << 31), EUNSUP, b"2^30"),
    (dict(ws=None), EINVAL, b"workspace"), (dict(bytes=8), EINVAL, b"workspace"), (dict(ws=ctypes.c_void_p(4100)), EINVAL, b"workspace"),
])
def test_probs_refuse(change, status, text):
    lib = yt.load()
    assert probs(lib, **change) == status
    assert text in lib.ythip_last_error()


def test_nothing_to_do():
    lib = yt.load()
    assert probs(lib, rows=0, x=None, p=None, ws=None) == 0 and probs(lib, n=0, x=None, p=None, ws=None) == 0
    assert verify(lib, B=0, target=None, tokens=None, ws=None) == 0
    assert lib.ythip_token_probs_workspace_size(0, 5) == 0 and lib.ythip_token_probs_workspace_size(1, 4096) == 0
    assert lib.ythip_token_probs_workspace_size(1, 151936) > 0 == lib.ythip_token_probs_workspace_size(256, 151936)


def verify(lib, **kw):
    i2 = _lib.i64array([1, 1])
    a = dict(dtype=_lib.F32, B=2, T=4, V=5000, target=FAKE, ts=i2, draft=None, ds=i2, tokens=FAKE, ldt=4, parents=None, ldp=4,
             tree_len=None, u=FAKE, ldu=4, u_next=FAKE, path=FAKE, ldpath=4, kept=FAKE, next=FAKE, ws=FAKE, bytes=1 << 20)
    a.update(kw)
    return lib.ythip_verify_drafts(*a.values(), None)


@pytest.mark.parametrize("change,status,text", [
    (dict(dtype=-1), EINVAL, b"dtype"), (dict(B=-1), EINVAL, b"negative"), (dict(T=0), EINVAL, b"tokens"),
    (dict(V=0), EINVAL, b"vocabulary"), (dict(T=1025, ldt=1025, ldu=1025, ldpath=1025), EUNSUP, b"1024"),
    (dict(V=(1 << 22) + 1), EUNSUP, b"vocabulary"), (dict(B=65536), EUNSUP, b"65535"), (dict(target=None), EINVAL, b"NULL"),
    (dict(tokens=None), EINVAL, b"NULL"), (dict(u=None), EINVAL, b"NULL"), (dict(u_next=None), EINVAL, b"NULL"),
    (dict(path=None), EINVAL, b"NULL"), (dict(kept=None), EINVAL, b"NULL"), (dict(next=None), EINVAL, b"NULL"),
    (dict(draft=FAKE, parents=FAKE), EINVAL, b"chain"), (dict(draft=FAKE, ds=None), EINVAL, b"strides"),
    (dict(ldt=3), EINVAL, b"strides"), (dict(ldu=3), EINVAL, b"strides"), (dict(ldpath=3), EINVAL, b"strides"),
    (dict(parents=FAKE, ldp=3), EINVAL, b"strides"), (dict(target=ctypes.c_void_p(4098)), EINVAL, b"within"),
    (dict(draft=ctypes.c_void_p(4098)), EINVAL, b"within"), (dict(ws=None), EINVAL, b"workspace"),
    (dict(bytes=63), EINVAL, b"workspace"), (dict(ws=ctypes.c_void_p(4100)), EINVAL, b"workspace"),
])
def test_verify_refuses(change, status, text):
    lib = yt.load()
    assert verify(lib, **change) == status
    assert text in lib.ythip_last_error()


def test_operators_take_device_tensors():
    x = torch.zeros(2, 3, 10)
    with pytest.raises(ValueError):
        yt.token_probs(x)
    with pytest.raises(ValueError):
        yt.verify_drafts(x, torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3), torch.zeros(2))


@pytest.mark.parametrize("draft", [False, True])
def test_the_model_draws_as_the_target_does(draft):
    """Over a grid of random numbers, the first token after the root is distributed as the target's row."""
    p, q = torch.tensor([0.5, 0.2, 0.3]), torch.tensor([0.2, 0.5, 0.3])
    n, count = 40, torch.zeros(3, dtype=torch.float64)
    grid = [(i + 0.5) / n for i in range(n)]
    if draft:
        target = torch.stack([p, p])[None]
        for x in range(3):
            for a in grid:
                for c in grid:
                    path, kept, nxt = model(target, torch.tensor([[0, x]]), torch.tensor([[0.0, a]]), torch.tensor([c]),
                                            draft=torch.stack([q, q])[None])
                    count[x if kept[0] == 2 else nxt[0]] += float(q[x]) / n ** 2
    else:
        target, tokens = torch.stack([p, p, p])[None], torch.tensor([[0, 2, 1]])
        for a in grid:
            for c in grid:
                path, kept, nxt = model(target, tokens, torch.tensor([[a, 0.0, 0.0]]), torch.tensor([c]), parents=torch.tensor([[-1, 0, 0]]))
                count[tokens[0, path[0][1]] if kept[0] == 2 else nxt[0]] += 1 / n ** 2
    assert torch.allclose(count, p.double(), atol=2 / n)
