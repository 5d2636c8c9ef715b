"""Attention over pages with a sliding window and sinks on the GPU, against window_ref (64 bits)."""
from __future__ import annotations

import math

import pytest
import torch

import ytensor_amd as yt
from window_ref import Rows, attention, compare

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cache(seed, lens, Hkv, page, d, dt, spare=3):
    """Pools of random rows and a table of scattered pages; what no sequence uses holds NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    k, v = (torch.randn(P, Hkv, page, d, generator=g).to(dt) for _ in range(2))
    perm = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), max(max(need), 1) + 1), -7, dtype=torch.int32)
    used, at = torch.zeros(P, page, dtype=torch.bool), 0
    for b, n in enumerate(lens):
        for c in range(need[b]):
            table[b, c] = perm[at]
            used[perm[at], :min(page, n - c * page)] = True
            at += 1
    k[~used[:, None].expand(-1, Hkv, -1)] = math.nan
    v[~used[:, None].expand(-1, Hkv, -1)] = math.nan
    return g, k.cuda(), v.cuda(), table.cuda(), ints(lens)


def tokens(g, B, Hq, Hkv, T, d, dt):
    return tuple(torch.randn(B, h, T, d, generator=g).to(dt).cuda() for h in (Hq, Hkv, Hkv))


def tree(g, B, T, far=5):
    back = torch.randint(1, far, (B, T), generator=g)
    return torch.clamp(torch.arange(T)[None] - back, min=-1).int().cuda()


WINDOWS = [(1, 0), (1, 3), (7, 1), (16, 0), (40, 17), (64, 64), (100, 4), (333, 0), (5000, 2), (60, 1000)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("T,kind", [(1, "chain"), (7, "tree"), (20, "chain"), (33, "tree"), (70, "chain"), (130, "tree"), (3, "none")])
@pytest.mark.parametrize("dtype,d,Hkv,G,page", [("bf16", 128, 2, 2, 16), ("f16", 64, 1, 5, 32), ("f32", 128, 1, 1, 64)])
def test_window(dtype, d, Hkv, G, page, T, kind, window, sinks):
    dt, lens = DT[dtype], [0, 1, 64, 700, 333]
    B = len(lens)
    g, kp, vp, table, kv_len = cache(T + window, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    if kind == "none":
        kn = vn = None
    parents = tree(g, B, T) if kind == "tree" else None
    tree_len = ints([max(0, T - b) for b in range(B)])
    out = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
    before = out.clone()
    yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents, tree_len=tree_len, out=out, window=window, sinks=sinks)
    want, tol = attention(q, kn, vn, Rows(kp, vp, table, kv_len), kv_len, parents, tree_len, window, sinks)
    compare(out, want, tol, before)


@pytest.mark.parametrize("dtype,B,Hkv,G,d,T,n,page,window,sinks", [
    ("bf16", 1, 2, 2, 128, 1, 40000, 64, 20000, 5), ("f16", 2, 1, 8, 128, 40, 9000, 16, 3000, 100),
    ("f32", 1, 1, 4, 64, 3, 20001, 1024, 9999, 0), ("bf16", 1, 1, 16, 64, 130, 5000, 32, 2047, 1),
    ("bf16", 3, 8, 2, 128, 4, 7001, 4096, 1025, 64), ("f32", 1, 2, 2, 128, 70, 3001, 32, 3000, 33),
    ("f16", 40, 1, 1, 64, 1, 777, 16, 50, 20), ("bf16", 70, 1, 1, 64, 2, 300, 16, 128, 0)])
def test_window_over_long_caches(dtype, B, Hkv, G, d, T, n, page, window, sinks):
    """The split and its merge, many row tiles, ragged batches."""
    dt = DT[dtype]
    lens = [n - (n - 5) * b // max(B - 1, 1) if B > 1 else n for b in range(B)]
    g, kp, vp, table, kv_len = cache(n, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    for parents in (None, tree(g, B, T)):
        out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents, scale=0.2, window=window, sinks=sinks)
        want, tol = attention(q, kn, vn, Rows(kp, vp, table, kv_len), kv_len, parents, None, window, sinks, scale=0.2)
        compare(out, want, tol)


@pytest.mark.parametrize("dtype,T,n,window,sinks,far", [
    ("bf16", 900, 0, 100, 4, 0), ("bf16", 900, 2, 100, 4, 0), ("f16", 700, 333, 64, 400, 0), ("f32", 300, 50, 17, 0, 0),
    ("bf16", 1100, 70, 1000, 90, 0), ("bf16", 600, 10, 30, 14, 2), ("f16", 400, 3, 20, 5, 3), ("f32", 300, 40, 100, 50, 2)])
def test_window_within_many_tokens(dtype, T, n, window, sinks, far):
    """Chunks and deep trees that are longer than the window, and sinks among the new tokens."""
    dt, B, Hkv, G, page, d = DT[dtype], 2, 1, 2, 32, 64
    g, kp, vp, table, kv_len = cache(T, [0, n], Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    parents = tree(g, B, T, far) if far else None
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents, window=window, sinks=sinks)
    want, tol = attention(q, kn, vn, Rows(kp, vp, table, kv_len), kv_len, parents, None, window, sinks)
    compare(out, want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,window,sinks", [(1, 30, 2), (9, 30, 2), (40, 20, 0), (140, 50, 3)])
def test_what_the_window_hides_never_reaches_a_row(dtype, T, window, sinks):
    """NaN and infinities in cached rows and new tokens that some queries see and others do not: those that do not are
    as without them."""
    dt, Hkv, G, page, d, n = DT[dtype], 1, 2, 16, 64, 200
    g, kp, vp, table, kv_len = cache(T, [n], Hkv, page, d, dt)
    q, kn, vn = tokens(g, 1, G, Hkv, T, d, dt)
    hit = n + 1 - window + min(T - 1, 3)  # hidden from token min(T - 1, 3) + 1 on
    rows = {hit - 1: math.nan, max(sinks, 5): math.inf, 100: math.nan}
    for r, x in rows.items():
        p = int(table[0, r // page])
        vp[p, 0, r % page, 3] = x
        if r != hit - 1:
            kp[p, 0, r % page, 5] = x
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, window=window, sinks=sinks)
    clean = Rows(torch.nan_to_num(kp, 0.0, 0.0, 0.0), torch.nan_to_num(vp, 0.0, 0.0, 0.0), table, kv_len)
    want, tol = attention(q, kn, vn, clean, kv_len, None, None, window, sinks)
    for t in range(T):
        sees = [r for r in rows if n + t - r < window or r < sinks]
        o = out[:, :, t].cpu()
        if not sees:
            compare(o, want[:, :, t], tol[:, :, t])
        else:
            assert sees == [hit - 1] and o[..., 3].isnan().all()
            keep = [i for i in range(d) if i != 3]
            compare(o[..., keep], want[:, :, t][..., keep], tol[:, :, t][..., keep])


def test_a_window_of_all_changes_nothing():
    """A window that reaches everything gives what no window gives, within two roundings of it, and window 0 its bits."""
    g, kp, vp, table, kv_len = cache(3, [500, 77], 2, 32, 128, torch.bfloat16)
    q, kn, vn = tokens(g, 2, 4, 2, 9, 128, torch.bfloat16)
    parents = tree(g, 2, 9)
    args = (q, kn, vn, kp, vp, table, kv_len)
    plain = yt.paged_attention(*args, parents=parents)
    assert torch.equal(yt.paged_attention(*args, parents=parents, window=0, sinks=9), plain)
    want, tol = attention(q, kn, vn, Rows(kp, vp, table, kv_len), kv_len, parents)
    for window in (600, 1 << 30, 1 << 40):
        compare(yt.paged_attention(*args, parents=parents, window=window, sinks=3), want, tol)
    with pytest.raises(ValueError):
        yt.paged_attention(*args, window=-1)
    with pytest.raises(ValueError):
        yt.paged_attention(*args, window=4, sinks=-1)


def test_rows_outside_the_window_are_not_read():
    """Pages that no token sees may have any id, and their sequences go on: a table whose middle is -1."""
    g, kp, vp, table, kv_len = cache(4, [4000, 1000], 2, 16, 64, torch.float16)
    q, kn, vn = tokens(g, 2, 4, 2, 3, 64, torch.float16)
    want, tol = attention(q, kn, vn, Rows(kp, vp, table, kv_len), kv_len, None, None, 200, 20)
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, window=200, sinks=20)
    compare(out, want, tol)
    table[0, 2:200], table[1, 2:40] = -1, 1 << 20
    assert torch.equal(yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, window=200, sinks=20), out)


def test_a_captured_window():
    """Lengths that grow between the replays of a graph."""
    g, kp, vp, table, kv_len = cache(5, [900, 640], 1, 32, 64, torch.bfloat16)
    q, kn, vn = tokens(g, 2, 4, 1, 2, 64, torch.bfloat16)
    need = yt.paged_workspace_bytes(torch.bfloat16, 2, 4, 1, 2, 64, table.shape[1], 32, window=128, sinks=4)
    out, ws = torch.empty_like(q), torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    call = lambda: yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, window=128, sinks=4, out=out, workspace=ws)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([900, 640], [1, 127], [128, 0], [511, 513]):
        kv_len.copy_(ints(lens))
        graph.replay()
        torch.cuda.synchronize()
        want, tol = attention(q, kn, vn, Rows(kp, vp, table, kv_len), kv_len, None, None, 128, 4)
        compare(out, want, tol)
