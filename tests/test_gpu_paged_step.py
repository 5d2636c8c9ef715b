"""The paged cache's calls as a server makes them, on the GPU: a pool that runs full, the documented step captured and
replayed, the views that a step has in hand."""
from __future__ import annotations

import pytest
import torch

import ytensor_amd as yt
from paged_ref import Pages, attention
from test_gpu_paged import DT, cache, compare, ints, tokens, tree

pytestmark = pytest.mark.gpu


def pools_of(g, L, P, Hkv, page, d, dt):
    k, v = (torch.randn(L, P, Hkv, page, d, generator=g).to(dt).cuda() for _ in range(2))
    return k, v, torch.randn(L, P, Hkv, d, generator=g).cuda()


def expect(pools, kn, vn, table, old, new, path=None):
    """What the append has to leave: the pools and, of each page written to, the sums (others as they were)."""
    k, v, sums = (x.cpu().clone() for x in pools)
    page, T, tol = k.shape[3], kn.shape[3], torch.zeros_like(sums, dtype=torch.float64)
    sums, table = sums.double(), torch.as_tensor(table)
    for b, (lo, hi) in enumerate(zip(old, new)):
        for i in range(hi - lo):
            f = -1 if i >= T else i if path is None else int(path[b, i])
            p, r = int(table[b, (lo + i) // page]), (lo + i) % page
            for pool, rows in ((k, kn), (v, vn)):
                pool[:, p, :, r] = rows[:, b, :, f].cpu() if 0 <= f < T else 0.0
        for c in range(lo // page, -(-hi // page) if hi > lo else 0):
            p, r = int(table[b, c]), min(page, hi - c * page)
            sums[:, p] = k[:, p, :, :r].double().sum(2)
            tol[:, p] = r * 2.0 ** -24 * k[:, p, :, :r].double().abs().sum(2)
    return k, v, sums, tol


def same(pools, want):
    assert torch.equal(pools[0].cpu(), want[0]) and torch.equal(pools[1].cpu(), want[1])
    assert ((pools[2].cpu().double() - want[2]).abs() <= want[3]).all()


@pytest.mark.parametrize("why", ["pool", "columns", "count"])
@pytest.mark.parametrize("dtype,page,d", [("bf16", 16, 64), ("f32", 64, 128), ("f16", 1024, 64)])
def test_append_after_a_refused_grow(dtype, page, d, why):
    """A sequence that the grow refuses keeps its rows, its pages' sums and its length, and no other sequence's page is
    touched, whatever ids stand behind its pages in the table."""
    dt, L, Hkv, T, columns = DT[dtype], 2, 2, page + 3, 4
    lens = [page + 5, 2 * page - 1, 3, 3 * page + 1, 0]
    n_new = [T, 1, T, page + 2 if why == "columns" else 2, 0]
    if why == "count":
        n_new[0] = -1
    need = [-(-n // page) for n in lens]
    P = sum(need) + (1 if why == "pool" else 9)
    g = torch.Generator().manual_seed(page)
    perm = torch.randperm(P, generator=g).tolist()
    used = perm[: sum(need)]
    table = torch.tensor(used)[torch.randint(0, len(used), (5, columns), generator=g)].int()  # live ids everywhere
    ref, at = torch.zeros(P, dtype=torch.int32), 0
    for b, n in enumerate(need):
        for c in range(n):
            table[b, c], ref[used[at]] = used[at], 1
            at += 1
    m = Pages(ref, table, torch.tensor(lens), page)
    m.grow(n_new)
    assert m.status == (yt.CACHE_ERR_INDEX if why == "count" else yt.CACHE_ERR_FULL)
    pools = pools_of(g, L, P, Hkv, page, d, dt)
    kn, vn = (torch.randn(L, 5, Hkv, T, d, generator=g).to(dt).cuda() for _ in range(2))
    want = expect(pools, kn, vn, m.table, lens, m.len)
    ref, table, old, status = ref.cuda(), table.cuda(), ints(lens), ints([0])
    new = torch.empty_like(old)
    yt.cache_grow(ref, table, old, ints(n_new), page, out=(ref, table, new), status=status)
    assert new.tolist() == m.len and table.tolist() == m.table
    yt.cache_append(kn, vn, *pools[:2], table, old, key_sums=pools[2], new_len=new, status=status)
    same(pools, want)
    assert status.item() == m.status


@pytest.mark.parametrize("page,T", [(16, 5), (16, 40), (128, 3)])
def test_append_of_more_rows_than_there_are(page, T):
    """Lengths that grew by more than the rows at hand: the rest are zeros, no row comes into use unwritten."""
    L, Hkv, d, lens = 2, 1, 64, [0, 7, page, 2 * page - 1]
    new = [T + 1, 7 + T + 3 * page, page + T, 2 * page - 1 + 4 * page]
    g = torch.Generator().manual_seed(T)
    columns = max(-(-n // page) for n in new)
    P = 4 * columns
    table = torch.randperm(P, generator=g).view(4, columns).int()
    pools = pools_of(g, L, P, Hkv, page, d, torch.bfloat16)
    kn, vn = (torch.randn(L, 4, Hkv, T, d, generator=g).bfloat16().cuda() for _ in range(2))
    path = torch.stack([torch.randperm(T, generator=g) for _ in lens]).int()
    path[2, 0] = T + 3
    want = expect(pools, kn, vn, table, lens, new, path)
    status = ints([0])
    yt.cache_append(kn, vn, *pools[:2], table.cuda(), ints(lens), path=path.cuda(), key_sums=pools[2], new_len=ints(new),
                    status=status)
    same(pools, want)
    assert status.item() == yt.CACHE_ERR_INDEX


def test_append_flags_what_it_leaves_out():
    """Lengths that shrank, pages outside the pool and rows past the table are left out and flagged; nothing else is."""
    g = torch.Generator().manual_seed(0)
    kn, vn = (torch.randn(1, 2, 1, 20, 64, generator=g).cuda() for _ in range(2))
    for table, old, new, bits, pages in (
            ([[0, 1], [2, 3]], [3, 0], [5, 4], 0, [0, 2]), ([[0, 1], [2, 3]], [3, 0], [2, 0], 1, []),
            ([[0, -1], [2, 3]], [10, 0], [20, 0], 1, [0]), ([[0, 1], [4, 3]], [0, 10], [0, 20], 1, [3]),
            ([[0, 1], [2, 3]], [30, 0], [33, 0], 1, [1]), ([[0, 1], [2, 3]], [-4, 0], [-4, 2], 0, [2]),
            ([[0, 1], [2, 3]], [-4, 0], [3, 2], 1, [2])):
        k, v = torch.zeros(1, 4, 1, 16, 64, device="cuda"), torch.zeros(1, 4, 1, 16, 64, device="cuda")
        status = ints([0])
        yt.cache_append(kn, vn, k, v, ints(table), ints(old), new_len=ints(new), status=status)
        assert status.item() == bits, (table, old, new)
        for pool in (k, v):
            assert (pool[0] != 0).flatten(1).any(1).nonzero().flatten().tolist() == pages, (table, old, new)


def test_append_takes_one_count():
    kn, kp = torch.zeros(1, 1, 1, 2, 64, device="cuda"), torch.zeros(1, 2, 1, 16, 64, device="cuda")
    args = (kn, kn, kp, kp.clone(), ints([[0]]), ints([0]))
    for bad in (dict(n_new=ints([1]), new_len=ints([1])), dict(n_new=ints([1]), status=ints([0])),
                dict(new_len=ints([1, 2])), dict(new_len=ints([1]).long()), dict(new_len=ints([1]), status=ints([0, 0]))):
        with pytest.raises(ValueError):
            yt.cache_append(*args, **bad)


@pytest.mark.parametrize("full", [False, True])
def test_the_documented_step_replayed(full):
    """The step as the integration notes give it, captured once: every replay adds its rows behind those of the one
    before, no page is lost, and a pool that runs full leaves the sequences as they were."""
    dt, L, B, Hq, Hkv, d, page, columns, T = torch.bfloat16, 2, 3, 4, 2, 64, 16, 8, 6
    P = 7 if full else 40
    g = torch.Generator().manual_seed(3)
    k_pool, v_pool, key_sums = pools_of(g, L, P, Hkv, page, d, dt)
    ref, status = torch.zeros(P, dtype=torch.int32, device="cuda"), ints([0])
    table, kv_len = torch.randint(0, P, (B, columns), generator=g).int().cuda(), ints([0] * B)
    old = torch.empty_like(kv_len)
    q = torch.empty(B, Hq, T, d, dtype=dt, device="cuda")
    k_all, v_all = (torch.empty(L, B, Hkv, T, d, dtype=dt, device="cuda") for _ in range(2))
    parents, path = torch.empty(B, T, dtype=torch.int32, device="cuda"), torch.empty(B, T, dtype=torch.int32, device="cuda")
    n_new, tree_len = ints([0] * B), ints([T] * B)
    rows = [[torch.zeros(L, Hkv, 0, d, dtype=dt) for _ in range(2)] for _ in range(B)]
    held = {}

    def fill(i):
        for t in (q, k_all, v_all):
            t.copy_(torch.randn(t.shape, generator=g).to(dt))
        parents.copy_(tree(g, B, T))
        path.copy_(torch.stack([torch.randperm(T, generator=g) for _ in range(B)]).int())
        n_new.copy_(torch.tensor([1 + (i + b) % T for b in range(B)], dtype=torch.int32))

    def step():
        held["o"] = [yt.paged_attention(q, k_all[l], v_all[l], k_pool[l], v_pool[l], table, kv_len, parents=parents,
                                        tree_len=tree_len) for l in range(L)]
        old.copy_(kv_len)
        yt.cache_grow(ref, table, kv_len, n_new, page, status=status)
        yt.cache_append(k_all, v_all, k_pool, v_pool, table, old, new_len=kv_len, path=path, key_sums=key_sums,
                        status=status)

    fill(0)
    keep = [x.clone() for x in (k_pool, v_pool, key_sums, ref, table, kv_len)]
    step()  # what the first calls set up is there before the capture
    for x, was in zip((k_pool, v_pool, key_sums, ref, table, kv_len), keep):
        x.copy_(was)
    status.zero_()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    m = Pages(ref, table, kv_len, page)
    for i in range(12):
        fill(i)
        before = list(m.len)
        torch.randn(1 << 20, device="cuda").sum().item()
        graph.replay()
        torch.cuda.synchronize()
        longest = max(max(before), 1)
        flat = [torch.zeros(B, Hkv, 256, d, dtype=dt) for _ in range(2)]
        for l in range(L):
            for b in range(B):
                for x in range(2):
                    flat[x][b, :, : before[b]] = rows[b][x][l]
            want, tol = attention(q, k_all[l], v_all[l], *flat, ints([[b] for b in range(B)]), ints(before), parents)
            compare(held["o"][l], want, tol)
        assert longest <= 256
        m.grow(n_new.tolist())
        for b in range(B):
            at = path[b, : m.len[b] - before[b]].tolist()
            for x, new in enumerate((k_all, v_all)):
                rows[b][x] = torch.cat([rows[b][x], new[:, b, :, at].cpu()], 2)
        assert kv_len.tolist() == m.len and ref.tolist() == m.ref and table.tolist() == m.table
        assert status.item() == m.status and sum(m.ref) == sum(m.pages(n) for n in m.len)
        for b in range(B):
            for c in range(m.pages(m.len[b])):
                p, r = m.table[b][c], min(page, m.len[b] - c * page)
                mine = rows[b][0][:, :, c * page: c * page + r]
                assert torch.equal(k_pool[:, p, :, :r].cpu(), mine)
                assert ((key_sums[:, p].cpu().double() - mine.double().sum(2)).abs()
                        <= r * 2.0 ** -24 * mine.double().abs().sum(2)).all()
    assert (m.status == yt.CACHE_ERR_FULL) == full


def test_views_with_one_sequence_or_token():
    """A dim of one element has no stride that matters, whatever the view says: slices of wider buffers whose width is
    no multiple of 16 bytes are taken, and written to, as they are."""
    dt, Hq, Hkv, d, page = torch.bfloat16, 4, 2, 64, 16
    g, kp, vp, table, kv_len = cache(2, [20], Hkv, page, d, dt)
    q, kn, vn = tokens(g, 1, Hq, Hkv, 1, d, dt)

    def odd(t):
        """t with strides of 1001 in its dims of one element"""
        st = [1001 if n == 1 else s for n, s in zip(t.shape, t.contiguous().stride())]
        return torch.empty_strided(t.shape, st, dtype=t.dtype, device="cuda").copy_(t)

    want, tol = attention(q, kn, vn, kp, vp, table, kv_len)
    out = odd(torch.zeros_like(q))
    yt.paged_attention(odd(q), odd(kn), odd(vn), kp, vp, table, kv_len, out=out)
    compare(out, want, tol)
    wide = torch.randn(1, (Hq + 2 * Hkv) * d + 3, generator=g).to(dt).cuda()  # a projection's row of odd width
    q, kn, vn = (x.unflatten(1, (-1, d))[:, :, None] for x in wide[:, :-3].split([Hq * d, Hkv * d, Hkv * d], 1))
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len)
    compare(yt.paged_attention(q, kn, vn, kp, vp, table, kv_len), want, tol)
    # one KV head, one layer: pools and rows with such strides
    g, kp, vp, table, kv_len = cache(2, [20], 1, page, d, dt)
    q, kn, vn = tokens(g, 1, 2, 1, 1, d, dt)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len)
    sums = torch.nan_to_num(kp.float()).sum(2)
    compare(yt.paged_attention(q, kn, vn, odd(kp), vp, table, kv_len), want, tol)
    out, _ = yt.paged_sparse_attention(q, kn, vn, kp, odd(vp), odd(sums), table, kv_len, 4)
    compare(out, want, tol)
    k2, v2, s2 = odd(kp[None]), vp[None].clone(), odd(sums[None])
    yt.cache_append(odd(kn[None]), vn[None], k2, v2, table, kv_len, key_sums=s2)
    assert torch.equal(k2[0, table[0, 1].long(), 0, 4], kn[0, 0, 0])
    assert torch.equal(v2[0, table[0, 1].long(), 0, 4], vn[0, 0, 0])
    held = k2[0, table[0, 1].long(), 0, :5].float()
    assert torch.allclose(s2[0, table[0, 1].long(), 0], held.sum(0), rtol=0, atol=5 * 2.0 ** -24 * held.abs().sum(0).max().item())
    pool = odd(torch.randn(1, 1, 3, 32, 64, generator=g).to(dt).cuda())  # one layer and one page, 2-byte elements
    yt.cache_copy_pages([pool], ints([0]), ints([0]))


def test_calls_with_nothing_to_do():
    """No tokens, no sequences, no columns, no pages."""
    kp = torch.zeros(1, 4, 1, 16, 64, device="cuda")
    for B, T, columns in ((0, 3, 2), (2, 0, 2), (2, 3, 0), (0, 0, 0)):
        kn = torch.zeros(1, B, 1, T, 64, device="cuda")
        table, lens = torch.zeros(B, columns, dtype=torch.int32, device="cuda"), ints([0] * B)
        yt.cache_append(kn, kn, kp, kp.clone(), table, lens)
        yt.cache_append(kn, kn, kp, kp.clone(), table, lens, new_len=lens.clone())
        assert (kp == 0).all()
        ref = ints([1, 0, 1, 1])
        r, t, n = yt.cache_grow(ref, table, lens, ints([0] * B), 16)
        assert r.tolist() == [1, 0, 1, 1] and n.tolist() == [0] * B
        yt.cache_free(ref, table, lens, ints([]), 16)
        yt.cache_fork([kp], ref, table, lens, ints([]), ints([]), 16)
        _, _, live = yt.cache_compact([kp], ref, table, lens, 16)
        assert live.item() == 3 and ref.tolist() == [1, 1, 1, 0]
    q, empty = torch.zeros(2, 2, 3, 64, device="cuda"), torch.zeros(0, 1, 16, 64, device="cuda")
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    assert (yt.paged_attention(q, None, None, empty, empty, none, ints([5, 0])) == 0).all()


def test_more_pieces_than_a_launch_holds():
    """4096 pairs in 4100 layers, each a workgroup's piece: all of them are copied."""
    L, n = 4100, 4096
    g = torch.Generator().manual_seed(12)
    pool = torch.randint(0, 2 ** 31 - 1, (L, 2 * n, 1), generator=g, dtype=torch.int32).cuda()
    order = torch.randperm(2 * n, generator=g).int().cuda()
    src, dst, was = order[:n], order[n:], pool.clone()
    yt.cache_copy_pages([pool], src, dst)
    assert torch.equal(pool[:, dst.long()], was[:, src.long()]) and torch.equal(pool[:, src.long()], was[:, src.long()])
    # the same as forks: each source has one row of its page, each gets the lowest free page
    pool.copy_(was)
    ref = torch.cat([torch.ones(n, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)]).cuda()
    table = torch.full((2 * n, 1), -1, dtype=torch.int32, device="cuda")
    table[:n, 0] = order[:n].argsort().int()  # page i of the first n, in some order
    kv_len = torch.cat([torch.ones(n, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)]).cuda()
    seqs = torch.arange(n, dtype=torch.int32, device="cuda")
    yt.cache_fork([pool], ref, table, kv_len, seqs, seqs + n, 16)
    assert (ref == 1).all() and (kv_len == 1).all() and torch.equal(table[n:, 0], seqs + n)
    assert torch.equal(pool[:, n:], was[:, table[:n, 0].long()]) and torch.equal(pool[:, :n], was[:, :n])


@pytest.mark.parametrize("lens,new", [([700], [130]), ([0, 900, 16], [130, 7, 0])])
def test_chunks_that_no_range_cuts(lens, new):
    """So many rows that every sequence stays whole: no workspace is asked for."""
    dt, B, T, Hkv, G, d = torch.bfloat16, len(lens), 130, 32, 8, 64
    g, k, v, table, kv_len = cache(7, lens, Hkv, 16, d, dt, columns=60)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    assert yt.paged_workspace_bytes(dt, B, Hkv * G, Hkv, T, d, 60, 16) == 0
    parents, tree_len = tree(g, B, T), ints(new)
    before = torch.full_like(q, 7.0)
    out = yt.paged_attention(q, kn, vn, k, v, table, kv_len, parents=parents, tree_len=tree_len, out=before.clone())
    compare(out, *attention(q, kn, vn, k, v, table, kv_len, parents, tree_len), before)
