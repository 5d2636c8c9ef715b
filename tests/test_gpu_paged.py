"""The paged cache's operators on the GPU against paged_ref (64 bits, plain Python)."""
from __future__ import annotations

import math

import pytest
import torch

import ytensor_amd as yt
from paged_ref import HALF_STEP, Pages, attention, select

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ints(x, dev="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def cache(seed, lens, Hkv, page, d, dt, spare=3, columns=None):
    """Pools of random rows and a table of scattered pages; what no sequence uses holds NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    columns = max(max(need), 1) + 1 if columns is None else columns
    k, v = (torch.randn(P, Hkv, page, d, generator=g).to(dt) for _ in range(2))
    perm = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), columns), -7, dtype=torch.int32)
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


def tree(g, B, T):
    back = torch.randint(1, 5, (B, T), generator=g)
    return torch.clamp(torch.arange(T)[None] - back, min=-1).int().cuda()


def compare(out, want, tol, before=None):
    """Every row that is computed within its bound; the others as they were."""
    o = out.detach().cpu().double()
    real = ~torch.isnan(want)
    assert torch.isfinite(o[real]).all()
    off = (o - want).abs()
    worst = (off[real] / tol[real].clamp(min=1e-300)).max().item() if real.any() else 0.0
    print(f"worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0
    if before is not None:
        assert torch.equal(out.cpu()[~real], before.cpu()[~real])


LENS = [[0], [1], [15, 16, 17], [300], [0, 64, 2049, 1]]


@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("T,kind", [(1, "chain"), (2, "tree"), (7, "tree"), (33, "chain"), (65, "tree"), (1, "none")])
@pytest.mark.parametrize("dtype,d,Hkv,G,page", [("bf16", 128, 2, 2, 16), ("f16", 64, 1, 5, 32), ("f32", 128, 2, 1, 64),
                                                 ("bf16", 64, 1, 17, 128), ("f32", 64, 1, 8, 16)])
def test_attention(dtype, d, Hkv, G, page, T, kind, lens):
    dt, B, Hq = DT[dtype], len(lens), Hkv * G
    g, kp, vp, table, kv_len = cache(len(lens) * 1000 + T, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hq, Hkv, T, d, dt)
    if kind == "none":
        kn = vn = None
    parents = tree(g, B, T) if kind == "tree" else None
    tree_len = ints([max(0, T - b) for b in range(B)]) if B > 1 else None
    out = torch.full((B, Hq, T, d), 7.0, dtype=dt, device="cuda")
    before = out.clone()
    yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents, tree_len=tree_len, out=out)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len, parents, tree_len)
    compare(out, want, tol, before)


@pytest.mark.parametrize("dtype,B,Hkv,G,d,T,n,page", [
    ("bf16", 1, 2, 2, 128, 1, 40000, 64), ("f16", 2, 1, 8, 128, 40, 9000, 16), ("f32", 1, 1, 4, 64, 3, 20001, 1024),
    ("bf16", 1, 1, 16, 64, 130, 5000, 32), ("bf16", 3, 8, 2, 128, 4, 7001, 4096), ("f32", 1, 2, 2, 128, 70, 3001, 32),
    ("f16", 40, 1, 1, 64, 1, 777, 16)])
def test_attention_over_long_caches(dtype, B, Hkv, G, d, T, n, page):
    """The split and its merge, many row tiles, ragged batches, the default out and a scale."""
    dt = DT[dtype]
    lens = [n - (n - 5) * b // max(B - 1, 1) if B > 1 else n for b in range(B)]
    g, kp, vp, table, kv_len = cache(n, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    parents = tree(g, B, T)
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents, scale=0.2)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len, parents, scale=0.2)
    compare(out, want, tol)


@pytest.mark.parametrize("dtype,B,T,columns", [("bf16", 150, 1, 40), ("f16", 70, 2, 20), ("f32", 129, 1, 9)])
def test_attention_of_many_sequences(dtype, B, T, columns):
    """More sequences than lanes of a wave, empty and full ones side by side, ranges that begin and end
    with a sequence."""
    dt, Hkv, page, d = DT[dtype], 1, 16, 64
    lens = [(0, 16 * columns, 64, 1, 128, 5)[b % 6] if b % 7 else 64 * (b % 3) for b in range(B)]
    lens = [min(n, 16 * columns) for n in lens]
    g, kp, vp, table, kv_len = cache(B, lens, Hkv, page, d, dt, columns=columns)
    q, kn, vn = tokens(g, B, 2, Hkv, T, d, dt)
    for new in ((kn, vn), (None, None)):
        want, tol = attention(q, *new, kp, vp, table, kv_len)
        compare(yt.paged_attention(q, *new, kp, vp, table, kv_len), want, tol)


@pytest.mark.parametrize("dtype,T,kind", [("bf16", 700, "tree"), ("f16", 1100, "chain"), ("f32", 300, "tree"),
                                          ("bf16", 4096, "tree")])
def test_attention_of_many_tokens(dtype, T, kind):
    """Long trees and chunks over several row tiles, with and without cached rows."""
    dt, B, Hkv, G, page, d = DT[dtype], 2, 1, 2, 32, 64
    g, kp, vp, table, kv_len = cache(T, [0, 333], Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    parents = tree(g, B, T) if kind == "tree" else None
    tree_len = ints([T - 3, T])
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents, tree_len=tree_len)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len, parents, tree_len)
    compare(out, want, tol, torch.zeros_like(out))


@pytest.mark.parametrize("dtype,lens,new", [
    ("bf16", [1500], [260]), ("bf16", [40, 2100], [260, 260]), ("f16", [0, 1900, 3], [7, 260, 0]),
    ("f32", [700, 0, 16, 900, 65], [1, 260, 64, 65, 0]), ("bf16", [0] * 7 + [1700], [0, 1, 260, 0, 3, 0, 0, 129]),
    ("f16", [400] * 9, [260] * 9)])
def test_attention_of_few_sequences_of_many_rows(dtype, lens, new):
    dt, B, T, Hkv, G = DT[dtype], len(lens), 260, 8, 4
    g, k, v, table, kv_len = cache(38, lens, Hkv, 16, 64, dt, columns=160)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, 64, dt)
    parents, tree_len = tree(g, B, T), ints(new)
    before = torch.full_like(q, 7.0)
    out = yt.paged_attention(q, kn, vn, k, v, table, kv_len, parents=parents, tree_len=tree_len, out=before.clone())
    compare(out, *attention(q, kn, vn, k, v, table, kv_len, parents, tree_len), before)


def test_attention_path_values():
    """A parent outside [0, child) ends the path, whatever it is."""
    dt, T, d = torch.float32, 9, 64
    g, kp, vp, table, kv_len = cache(8, [20], 1, 16, d, dt)
    q, kn, vn = tokens(g, 1, 2, 1, T, d, dt)
    parents = ints([[5, 0, 2, 7, -2 ** 31, 2 ** 31 - 1, 1, 6, 100]])
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len, parents)
    compare(out, want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_strides_and_layouts(dtype):
    """Rows of a fused projection, pools [P, page, Hkv, d], a table with a longer row stride, out
    over [B, T, Hq, d]."""
    dt, B, Hq, Hkv, T, d, page = DT[dtype], 2, 6, 2, 5, 128, 32
    g, kp, vp, table, kv_len = cache(3, [70, 33], Hkv, page, d, dt)
    wide = torch.randn(B, T, (Hq + 2 * Hkv) * d, generator=g).to(dt).cuda().view(B, T, Hq + 2 * Hkv, d).transpose(1, 2)
    q, kn, vn = wide[:, :Hq], wide[:, Hq:Hq + Hkv], wide[:, Hq + Hkv:]
    kp2, vp2 = (p.transpose(1, 2).contiguous().transpose(1, 2) for p in (kp, vp))
    table2 = torch.cat([table, table], 1)[:, :table.shape[1]]
    out = torch.empty(B, T, Hq, d, dtype=dt, device="cuda").transpose(1, 2)
    yt.paged_attention(q, kn, vn, kp2, vp2, table2, kv_len, out=out)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len)
    compare(out, want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_keeps_to_the_path(dtype, bad):
    """K and V of a sibling branch, of rows past the length and past tree_len never reach a row; on
    the row's own path they do, as in the formula."""
    dt, B, Hq, Hkv, T, d, page = DT[dtype], 2, 4, 2, 40, 64, 16
    g, kp, vp, table, kv_len = cache(5, [37, 100], Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hq, Hkv, T, d, dt)
    parents = tree(g, B, T)
    parents[:, 3:6] = ints([0, 0, 1])  # 3: leaf of its own
    parents[:, 6:] = torch.clamp(parents[:, 6:], min=4)
    tree_len = ints([T, T - 2])
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len, parents, tree_len)
    kn2, vn2 = kn.clone(), vn.clone()
    kn2[:, :, 3], vn2[:, :, 3] = bad, bad
    kn2[1, :, T - 2:], vn2[1, :, T - 2:] = bad, bad
    out = yt.paged_attention(q, kn2, vn2, kp, vp, table, kv_len, parents=parents, tree_len=tree_len)
    own = torch.zeros_like(want, dtype=torch.bool)
    own[:, :, 3] = True
    o = out.cpu().double()
    want[own] = math.nan
    compare(torch.where(own, 0.0, o), want, tol)
    vn3 = vn.clone()
    vn3[:, :, 3, ::2] = bad  # V alone: the row itself gets what p . V gives, the others nothing
    out = yt.paged_attention(q, kn, vn3, kp, vp, table, kv_len, parents=parents, tree_len=tree_len)
    o = out.cpu().double()
    compare(torch.where(own, 0.0, o), want, tol)
    odd = o[:, :, 3]
    assert torch.isfinite(odd[..., 1::2]).all()
    assert (torch.isnan(odd[..., ::2]).all() if math.isnan(bad) else (odd[..., ::2] == bad).all())


def test_attention_bad_pages_and_lengths():
    """Ids outside the pool hide their rows; lengths are clamped to what the table can hold."""
    dt, page, d = torch.bfloat16, 16, 128
    g, kp, vp, table, kv_len = cache(11, [100, 64, 48, 5], 2, page, d, dt, columns=7)
    q, kn, vn = tokens(g, 4, 4, 2, 3, d, dt)
    table[0, 2], table[0, 5], table[1, 0] = -1, kp.shape[0], 2 ** 31 - 1
    table[2, :] = -5
    kv_len[3] = -4
    for new in ((kn, vn), (None, None)):
        out = yt.paged_attention(q, *new, kp, vp, table, kv_len)
        want, tol = attention(q, *new, kp, vp, table, kv_len)
        compare(out, want, tol)
    kp, vp = torch.nan_to_num(kp), torch.nan_to_num(vp)
    table[0] = ints([1, 2, 3, 4, 5, 6, 7])
    kv_len[0] = 2 ** 31 - 1
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len)
    compare(out, want, tol)


def test_attention_large_scores():
    """Scores far apart, all -inf, and a huge scale: the running maximum follows, nothing overflows."""
    dt, page, d = torch.float32, 16, 64
    g, kp, vp, table, kv_len = cache(12, [400], 1, page, d, dt)
    q, kn, vn = tokens(g, 1, 2, 1, 4, d, dt)
    q *= 30
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, scale=-3.0)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len, scale=-3.0)
    compare(out, want, tol)
    q = torch.ones_like(q)
    kp[:], kn[:] = -math.inf, -math.inf
    out = yt.paged_attention(q, kn, torch.ones_like(vn), kp, torch.ones_like(vp), table, kv_len)
    assert (out == 0).all()
    kn[:] = math.nan
    assert torch.isnan(yt.paged_attention(q, kn, vn, kp, torch.ones_like(vp), table, kv_len)).all()


def test_attention_offsets_past_32_bits():
    """Pages that lie more than 2^32 bytes and 2^31 elements into the pool."""
    P, Hkv, page, d = 40000, 8, 64, 128   # 2.6e9 elements, 5.2 GB
    kp = torch.empty(P, Hkv, page, d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(1)
    at = [P - 1, 3, P - 2, 33000]
    small = [torch.randn(4, Hkv, page, d, generator=g).bfloat16().cuda() for _ in range(2)]
    kp[at] = small[0]
    vp = torch.empty_like(kp)
    vp[at] = small[1]
    q, kn, vn = tokens(g, 1, 16, Hkv, 2, d, torch.bfloat16)
    out = yt.paged_attention(q, kn, vn, kp, vp, ints([at]), ints([250]))
    want, tol = attention(q, kn, vn, *small, ints([[0, 1, 2, 3]]), ints([250]))
    compare(out, want, tol)
    ref = torch.ones(P, dtype=torch.int32, device="cuda")
    pools = [kp[None], vp[None]]
    yt.cache_copy_pages(pools, ints([P - 1, 33000]), ints([7, 39990]))
    assert torch.equal(kp[7], small[0][0]) and torch.equal(vp[39990], small[1][3])


@pytest.mark.parametrize("dtype,B,Hkv,G,d,T,page,lens,top", [
    ("bf16", 1, 2, 2, 128, 1, 16, [777], 5), ("f16", 3, 1, 5, 64, 4, 32, [0, 31, 2000], 8),
    ("f32", 2, 2, 4, 128, 3, 64, [64, 1000], 3), ("bf16", 2, 1, 1, 64, 9, 16, [500, 16], 1),
    ("f16", 1, 4, 16, 128, 2, 128, [9000], 40), ("bf16", 1, 1, 2, 128, 1, 16, [20000], 600),
    ("f32", 1, 1, 20, 64, 2, 16, [300], 64)])
@pytest.mark.parametrize("kind", ["chain", "tree", "none"])
def test_sparse(dtype, B, Hkv, G, d, T, page, lens, top, kind):
    dt = DT[dtype]
    g, kp, vp, table, kv_len = cache(T + top, lens, Hkv, page, d, dt)
    sums = torch.nan_to_num(kp.float()).sum(2)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    parents, tree_len = None, None
    if kind == "tree":
        parents, tree_len = tree(g, B, T), ints([max(0, T - 2 * b) for b in range(B)])
    if kind == "none":
        kn = vn = None
    out = torch.full((B, Hkv * G, T, d), 7.0, dtype=dt, device="cuda")
    before = out.clone()
    _, sel = yt.paged_sparse_attention(q, kn, vn, kp, vp, sums, table, kv_len, top, parents=parents,
                                       tree_len=tree_len, out=out)
    want_sel = select(q, sums, table, kv_len, page, top, tree_len)
    assert torch.equal(sel.cpu(), want_sel)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len, parents, tree_len, sel=want_sel)
    compare(out, want, tol, before)


def test_sparse_ties_nan_and_bad_pages():
    """Equal scores (of both zeros too) go to the lower column, NaN is the lowest, a page id outside
    the pool has no score and no rows."""
    page, d, n = 16, 64, 1024
    g, kp, vp, table, kv_len = cache(4, [n * page - 3], 1, page, d, torch.bfloat16)
    sums = torch.zeros(kp.shape[0], 1, d, device="cuda")
    at = table[0, :n].long()
    sums[at[3::7]] = -0.0
    sums[at[700]] = math.nan
    sums[at[10::100]] = 1.0
    sums[at[200], 0, 5] = math.inf
    sums[at[201], 0, 5] = -math.inf
    table[0, 30] = -1
    q, kn, vn = tokens(g, 1, 2, 1, 2, d, torch.bfloat16)
    q = q.abs()
    for top in (1, 2, 5, 64, 1000, 1023, 1024, 1500):
        _, sel = yt.paged_sparse_attention(q, kn, vn, kp, vp, sums, table, kv_len, top)
        want = select(q, sums, table, kv_len, page, top)
        assert torch.equal(sel.cpu(), want), top


@pytest.mark.parametrize("n,columns", [(1500, 1500), (900, 1000), (9000, 9001)])
def test_sparse_choice_of_few_of_many(n, columns):
    """Both sizes of the choosing workgroup, ranks kept and read again, scores alike in their first bits."""
    page, d = 16, 64
    g = torch.Generator().manual_seed(n)
    kp = torch.randn(64, 1, page, d, generator=g).bfloat16().cuda()
    table = torch.randint(0, 64, (1, columns), generator=g).int().cuda()
    sums = 1 + 1e-6 * torch.randn(64, 1, d, generator=g).cuda()
    q = torch.rand(1, 2, 3, d, generator=g).bfloat16().cuda()
    for top in (1, 7, 100, min(n - 1, 4096)):
        out, sel = yt.paged_sparse_attention(q, None, None, kp, kp, sums, table, ints([n * page]), top)
        assert torch.equal(sel.cpu(), select(q, sums, table, ints([n * page]), page, top))


def test_sparse_many_columns():
    """The widest table."""
    page, d, n = 16, 64, 65536
    kp = torch.randn(64, 1, page, d, device="cuda", dtype=torch.bfloat16)
    vp = torch.randn_like(kp)
    g = torch.Generator().manual_seed(2)
    table = torch.randint(0, 64, (1, n), generator=g).int().cuda()
    sums = kp.float().sum(2)
    kv_len = ints([n * page - 20])
    q, kn, vn = tokens(g, 1, 1, 1, 1, d, torch.bfloat16)
    out, sel = yt.paged_sparse_attention(q, kn, vn, kp, vp, sums, table, kv_len, 1500)
    want_sel = select(q, sums, table, kv_len, page, 1500)
    assert torch.equal(sel.cpu(), want_sel)
    want, tol = attention(q, kn, vn, kp, vp, table, kv_len, sel=want_sel)
    compare(out, want, tol)


# ------------------------------------------------------------- rows and pages

@pytest.mark.parametrize("dtype,d,page", [("bf16", 128, 64), ("f16", 64, 16), ("f32", 128, 32), ("bf16", 8, 16),
                                          ("f32", 1024, 16), ("f16", 96, 16)])
@pytest.mark.parametrize("T,how", [(1, "all"), (5, "path"), (100, "all"), (33, "some")])
def test_append(dtype, d, page, T, how):
    dt, L, Hkv, lens = DT[dtype], 2, 3, [0, 15, 16, 70]
    B = len(lens)
    g = torch.Generator().manual_seed(T)
    columns = -(-(max(lens) + T) // page) + 1
    P = B * columns + 2
    kp, vp = (torch.randn(L, P, Hkv, page, d, generator=g).to(dt).cuda() for _ in range(2))
    kn, vn = (torch.randn(L, B, Hkv, T, d, generator=g).to(dt).cuda() for _ in range(2))
    table = torch.randperm(P, generator=g)[:B * columns].view(B, columns).int().cuda()
    sums = torch.full((L, P, Hkv, d), 3.0, device="cuda")
    n_new = path = None
    if how != "all":
        n_new = ints([T, 0, 3, -2] if how == "some" else [2, 5, 9, 1])
    if how == "path":
        path = torch.stack([torch.randperm(T, generator=g) for _ in range(B)]).int().cuda()
        path[0, 1] = T  # no such row
        path[1, 2] = -1
    want = [kp.cpu().clone(), vp.cpu().clone(), sums.cpu().double()]
    tol = torch.zeros_like(want[2])
    for b, n in enumerate(lens):
        more = T if n_new is None else max(0, min(int(n_new[b]), T))
        for i in range(more):
            f = i if path is None else int(path[b, i])
            for pool, new in ((want[0], kn), (want[1], vn)):
                row = new[:, b, :, f].cpu() if 0 <= f < T else torch.zeros(L, Hkv, d, dtype=dt)
                pool[:, int(table[b, (n + i) // page]), :, (n + i) % page] = row
        for c in range(n // page, -(-(n + more) // page) if more else 0):
            p, r = int(table[b, c]), min(page, n + more - c * page)
            rows = want[0][:, p, :, :r].double()
            want[2][:, p] = rows.sum(2)
            tol[:, p] = r * 2.0 ** -24 * rows.abs().sum(2)
    yt.cache_append(kn, vn, kp, vp, table, ints(lens), n_new=n_new, path=path, key_sums=sums)
    assert torch.equal(kp.cpu(), want[0]) and torch.equal(vp.cpu(), want[1])
    assert ((sums.cpu().double() - want[2]).abs() <= tol).all()
    again = sums.clone()
    yt.cache_append(kn, vn, kp, vp, table, ints(lens), n_new=n_new, path=path, key_sums=sums)
    assert torch.equal(again, sums)


def test_append_out_of_range():
    """Pages outside the pool, rows past the table and negative lengths are not written."""
    kp = torch.zeros(1, 4, 1, 16, 64, device="cuda")
    vp, kn = torch.zeros_like(kp), torch.ones(1, 3, 1, 40, 64, device="cuda")
    table = ints([[0, -1, 1], [2, 9, 3], [0, 0, 0]])
    yt.cache_append(kn, kn, kp, vp, table, ints([10, 40, -1]))
    used = (kp[0, :, 0, :, 0] != 0).cpu()
    assert used.sum(1).tolist() == [6, 16, 0, 8] and torch.equal(kp, vp)


def state(seed, B, columns, P, page, lens, share=()):
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(P, generator=g).tolist()
    table, ref = torch.randint(-3, P, (B, columns), generator=g).int(), torch.zeros(P, dtype=torch.int32)
    for b, n in enumerate(lens):
        for c in range(-(-n // page)):
            table[b, c] = perm.pop()
    for a, b in share:
        table[b, 0] = table[a, 0]
    for b, n in enumerate(lens):
        for c in range(-(-n // page)):
            ref[table[b, c]] += 1
    return g, ref.cuda(), table.cuda(), ints(lens)


def pools_of(g, L, P, page):
    return [torch.randn(L, P, 2, page, 64, generator=g).bfloat16().cuda(),
            torch.randn(L, P, 3, 1, generator=g).cuda(),                      # 12-byte pages
            torch.randn(L, P, 1, page, 512, generator=g).cuda().transpose(0, 0)]


def both(call, m, ref, table, kv_len, pools, status):
    """In place and into other arrays: the same arrays as the model's."""
    held = [t.clone() for t in (ref, table, kv_len)]
    backup = [p.clone() for p in pools]
    into = tuple(torch.full_like(t, -99) for t in held)
    for out in (into, None):
        for p, q in zip(pools, backup):
            p.copy_(q)
        status.zero_()
        got = call(*held, out, status)
        assert [x.tolist() for x in got[:3]] == [m.ref, m.table, m.len] and status.item() == m.status
        if out is not None:
            assert all(torch.equal(a, b) for a, b in zip(held, (ref, table, kv_len)))
        for p, want in zip(pools, m.pools):
            assert torch.equal(p.cpu(), want)


@pytest.mark.parametrize("P,B", [(40, 5), (9000, 70), (20000, 1500)])
@pytest.mark.parametrize("scarce", [False, True])
def test_grow(P, B, scarce):
    page, columns = 16, 24
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, min(60, 16 * (P // B - 1)), (B,), generator=g).tolist()
    g, ref, table, kv_len = state(P, B, columns, P, page, lens)
    n_new = torch.randint(0, 300 if scarce else max(1, 16 * ((P // B) - 4)), (B,), generator=g).tolist()
    n_new[1], n_new[-1] = -1, 0
    n_new[2] = 16 * columns - lens[2] + (1 if B > 5 else 0)
    m = Pages(ref, table, kv_len, page)
    m.grow(n_new)
    both(lambda r, t, n, out, st: yt.cache_grow(r, t, n, ints(n_new), page, out=out, status=st), m, ref, table, kv_len,
         [], ints([0]))


@pytest.mark.parametrize("L,page", [(1, 16), (3, 64)])
@pytest.mark.parametrize("spare", [0, 2, 30])
def test_fork(L, page, spare):
    lens = [page * 3, page * 2 + 5, 1, 0, 0, 0, 0, 0, 0, 0, 0, page - 1]
    P = 3 + 3 + 1 + 1 + spare
    g, ref, table, kv_len = state(page, len(lens), 4, P, page, lens)
    pools = pools_of(g, L, P, page)
    table[1, 1] = P + 2  # an id outside the pool is passed on, no count touched
    src, dst = [1, 0, 1, 11, 4, 2, 9, 12, 0, 2, 3], [3, 4, 5, 3, 6, 0, 7, 8, -1, 8, 9]
    m = Pages(ref, table, kv_len, page, pools)
    m.fork(src, dst)
    both(lambda r, t, n, out, st: yt.cache_fork(pools, r, t, n, ints(src), ints(dst), page, out=out, status=st), m, ref,
         table, kv_len, pools, ints([0]))


def test_fork_many():
    """More pairs than the deciding workgroup has threads."""
    page, B, n, P = 16, 4000, 1900, 6000
    lens = [17 + i % 16 for i in range(n)] + [0] * (B - n)
    g, ref, table, kv_len = state(1, B, 3, P, page, lens)
    src = torch.randint(0, n, (n,), generator=g).tolist()
    dst = (n + torch.randperm(B - n, generator=g)[:n]).tolist()
    m = Pages(ref, table, kv_len, page)
    m.fork(src, dst)
    both(lambda r, t, k, out, st: yt.cache_fork([], r, t, k, ints(src), ints(dst), page, out=out, status=st), m, ref,
         table, kv_len, [], ints([0]))


@pytest.mark.parametrize("seqs", [[0], [3, 1, 3, 0, 3], [2, 2, -1, 6, 4, 5], []])
def test_free(seqs):
    page, lens = 16, [40, 33, 0, 64, 16, 7]
    g, ref, table, kv_len = state(8, 6, 5, 20, page, lens, share=[(0, 1), (0, 3)])
    table[5, 0] = 20
    kv_len[2] = 0
    m = Pages(ref, table, kv_len, page)
    m.free(seqs)
    both(lambda r, t, n, out, st: yt.cache_free(r, t, n, ints(seqs), page, out=out, status=st), m, ref, table, kv_len,
         [], ints([0]))


@pytest.mark.parametrize("P,B,L", [(12, 2, 1), (40, 5, 2), (5000, 60, 1), (9000, 400, 1)])
def test_compact(P, B, L):
    page, columns = 16, 8
    g = torch.Generator().manual_seed(P)
    lens = torch.randint(0, min(120, 16 * (P // B)), (B,), generator=g).tolist()
    g, ref, table, kv_len = state(P + 1, B, columns, P, page, lens, share=[(0, 1)] if min(lens[:2]) > 0 else [])
    pools = pools_of(g, L, P, page)[:3 if P < 100 else 2]
    m = Pages(ref, table, kv_len, page, pools)
    live = m.compact()

    def call(r, t, n, out, st):
        r2, t2, got = yt.cache_compact(pools, r, t, n, page, out=None if out is None else out[:2])
        assert got.tolist() == [live]
        return r2, t2, n
    both(call, m, ref, table, kv_len, pools, ints([0]))
    assert live == sum(r > 0 for r in m.ref[:live])


def test_copy_pages():
    g = torch.Generator().manual_seed(3)
    pools = pools_of(g, 2, 10, 16)
    want = [p.clone() for p in pools]
    src, dst, st = ints([1, 2, 10, 3, 1]), ints([4, 5, 6, -1, 7]), ints([0])
    yt.cache_copy_pages(pools, src, dst, status=st)
    for p, w in zip(pools, want):
        w[:, [4, 5, 7]] = w[:, [1, 2, 1]]
        assert torch.equal(p, w)
    assert st.item() == yt.CACHE_ERR_INDEX


def test_refusals_of_the_python_layer():
    g, kp, vp, table, kv_len = cache(1, [20, 3], 2, 16, 64, torch.bfloat16)
    q, kn, vn = tokens(g, 2, 4, 2, 3, 64, torch.bfloat16)
    ok = dict(q=q, k_new=kn, v_new=vn, k_pool=kp, v_pool=vp, table=table, kv_len=kv_len)
    for bad in (dict(q=q[0]), dict(q=q[:, :3]), dict(q=q.float()), dict(k_new=None), dict(k_new=kn[:, :, :2]),
                dict(v_pool=vp[:3]), dict(k_pool=kp.transpose(2, 3)), dict(table=table[:1]), dict(table=table.long()),
                dict(kv_len=kv_len.long()), dict(kv_len=kv_len.cpu()), dict(parents=table[:, :2]), dict(tree_len=kv_len[:1]),
                dict(out=q[:, :2]), dict(table=table.t().contiguous().t()),
                dict(k_pool=kp[:, :, :15], v_pool=vp[:, :, :15]), dict(k_pool=kp[..., :32], v_pool=vp[..., :32])):
        with pytest.raises((ValueError, yt.YthipError)):
            yt.paged_attention(**{**ok, **bad})
    with pytest.raises(ValueError):
        yt.paged_sparse_attention(**ok, key_sums=kp.sum(2), top_k=2)
    ref = torch.zeros(kp.shape[0], dtype=torch.int32, device="cuda")
    for bad in (dict(n_new=kv_len[:1]), dict(ref=ref.long()), dict(status=kv_len), dict(out=(ref, table, ref)),
                dict(page=17)):
        with pytest.raises((ValueError, yt.YthipError)):
            yt.cache_grow(**{**dict(ref=ref, table=table, kv_len=kv_len, n_new=kv_len, page=16), **bad})
    with pytest.raises(ValueError):
        yt.cache_fork([kp[None].transpose(2, 3)], ref, table, kv_len, kv_len, kv_len, 16)
    with pytest.raises(ValueError):
        yt.cache_append(kn[None], vn[None], kp, vp, table, kv_len)


# ------------------------------------------------------------------- together

def test_refusals_of_expanded_arguments():
    """A table whose rows are one row (stride 0), and a workspace of fewer bytes than elements."""
    g, k, v, table, kv_len = cache(5, [900, 900], 2, 16, 64, torch.bfloat16, columns=57)
    q, kn, vn = tokens(g, 2, 4, 2, 1, 64, torch.bfloat16)
    with pytest.raises(yt.YthipError, match="stride"):
        yt.paged_attention(q, kn, vn, k, v, table[:1].expand(2, 57), kv_len)
    with pytest.raises(yt.YthipError, match="stride"):
        yt.cache_free(torch.ones(8, dtype=torch.int32, device="cuda"), table[:1].expand(2, 57), kv_len, ints([0]), 16)
    space = torch.empty(1, dtype=torch.uint8, device="cuda").expand(1 << 26)
    with pytest.raises(ValueError, match="contiguous"):
        yt.paged_attention(q, kn, vn, k, v, table, kv_len, workspace=space)


@pytest.mark.parametrize("apart", range(8))
@pytest.mark.parametrize("columns", [12, 700])
def test_some_outputs_in_place(columns, apart):
    """Any of ref, table and kv_len written in place and the others elsewhere: the same state."""
    _, ref, table, kv_len = state(61, 40, columns, 600, 16, [(7 * b) % 150 for b in range(30)] + [0] * 10)
    n_new = [b % 20 for b in range(38)] + [0, 0]
    want, got = [], []
    for outs, bits in ((want, 0), (got, apart)):
        st = [x.clone() for x in (ref, table, kv_len)]
        for call in (lambda o: yt.cache_grow(*st, ints(n_new), 16, out=o),
                     lambda o: yt.cache_fork((), *st, ints([3, 4]), ints([39, 38]), 16, out=o),
                     lambda o: yt.cache_free(*st, ints([0, 5, 39]), 16, out=o)):
            o = tuple(torch.full_like(x, 77) if bits >> i & 1 else x for i, x in enumerate(st))
            call(o)
            st = list(o)
            outs += [x.cpu() for x in st]
    assert all(torch.equal(x, y) for x, y in zip(want, got)) and want[5][39] == want[2][3] > 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_generation_with_drafts(dtype):
    """Prompt, fork, drafted trees verified and committed, sparse attention, an end and a packing:
    after every step the attention over the pages is that over each sequence's rows side by side."""
    dt, L, B, Hq, Hkv, d, page, P, columns, T = DT[dtype], 2, 4, 4, 2, 64, 16, 40, 8, 6
    g = torch.Generator().manual_seed(9)
    kp, vp = (torch.full((L, P, Hkv, page, d), math.nan, device="cuda").to(dt) for _ in range(2))
    sums = torch.zeros(L, P, Hkv, d, device="cuda")
    ref, status = torch.zeros(P, dtype=torch.int32, device="cuda"), ints([0])
    table, kv_len = torch.full((B, columns), -1, dtype=torch.int32, device="cuda"), ints([0] * B)
    rows = [[torch.zeros(L, Hkv, 0, d, dtype=dt) for _ in range(2)] for _ in range(B)]  # each sequence's K, V

    def new(n):
        return tuple(torch.randn(L, B, Hkv, n, d, generator=g).to(dt).cuda() for _ in range(2))

    def commit(kn, vn, n_new, path=None):
        old = kv_len.clone()
        yt.cache_grow(ref, table, kv_len, ints(n_new), page, status=status)
        yt.cache_append(kn, vn, kp, vp, table, old, n_new=ints(n_new), path=path, key_sums=sums)
        for b, n in enumerate(n_new):
            at = list(range(n)) if path is None else path[b, :n].tolist()
            for i, t in enumerate((kn, vn)):
                rows[b][i] = torch.cat([rows[b][i], t[:, b, :, at].cpu()], 2)

    def look(kn, vn, parents=None, tree_len=None):
        q = torch.randn(B, Hq, kn.shape[3], d, generator=g).to(dt).cuda()
        longest = max(r[0].shape[2] for r in rows)
        flat = [torch.zeros(B, Hkv, 32768, d, dtype=dt) for _ in range(2)]
        for b in range(B):
            for i in range(2):
                flat[i][b, :, :rows[b][i].shape[2]] = rows[b][i][1]
        assert kv_len.tolist() == [r[0].shape[2] for r in rows] and longest < 32768
        out = yt.paged_attention(q, kn[1], vn[1], kp[1], vp[1], table, kv_len, parents=parents, tree_len=tree_len)
        side = ints([[b] for b in range(B)])
        want, tol = attention(q, kn[1], vn[1], *flat, side, kv_len, parents, tree_len)
        compare(out, want, tol)
        o2, sel = yt.paged_sparse_attention(q, kn[1], vn[1], kp[1], vp[1], sums[1], table, kv_len, columns,
                                            parents=parents, tree_len=tree_len)
        compare(o2, want, tol)
        _, sel = yt.paged_sparse_attention(q, kn[1], vn[1], kp[1], vp[1], sums[1], table, kv_len, 2, parents=parents,
                                           tree_len=tree_len)
        assert torch.equal(sel.cpu(), select(q, sums[1], table, kv_len, page, 2, tree_len))

    k, v = new(37)
    look(k, v)
    commit(k, v, [37, 20, 0, 0])
    yt.cache_fork([kp, vp, sums], ref, table, kv_len, ints([0, 1]), ints([2, 3]), page, status=status)
    rows[2], rows[3] = [list(r) for r in (rows[0], rows[1])]
    for _ in range(3):
        k, v = new(T)
        parents = tree(g, B, T)
        look(k, v, parents, ints([T, T - 1, T, 1]))
        path = torch.zeros(B, T, dtype=torch.int32)
        for b in range(B):
            path[b, :2] = torch.tensor([0, 1 + b % 3])
        commit(k, v, [2, 1, 2, 1], path.cuda())
    yt.cache_free(ref, table, kv_len, ints([0]), page, status=status)
    rows[0] = [torch.zeros(L, Hkv, 0, d, dtype=dt) for _ in range(2)]
    look(*new(2))
    _, _, live = yt.cache_compact([kp, vp, sums], ref, table, kv_len, page)
    assert live.item() == len({p for b in range(B) for p in table[b, :-(-int(kv_len[b]) // page)].tolist()})
    assert (ref[:live.item()] > 0).all() and (ref[live.item():] == 0).all() and status.item() == 0
    look(*new(1))


def test_a_captured_step():
    """Attend, sparse attend, grow and append captured as one graph and replayed with other work
    between: every replay gives what the calls give one by one."""
    dt, B, Hq, Hkv, d, page, P, columns, T = torch.bfloat16, 3, 4, 2, 128, 16, 60, 12, 2
    g = torch.Generator().manual_seed(4)
    _, k1, v1, table0, len0 = cache(6, [50, 17, 0], Hkv, page, d, dt, spare=P, columns=columns)
    P = k1.shape[0]
    ref0 = torch.zeros(P, dtype=torch.int32, device="cuda")
    for b, n in enumerate(len0.tolist()):
        ref0[table0[b, :-(-n // page)].long()] = 1
    q, kn, vn = tokens(g, B, Hq, Hkv, T, d, dt)

    def fresh():
        kp, vp = k1.clone()[None], v1.clone()[None]
        return dict(kp=kp, vp=vp, sums=torch.nan_to_num(kp.float()).sum(3), ref=ref0.clone(), table=table0.clone(),
                    len=len0.clone(), old=len0.clone(), n=ints([2, 1, 2]))

    def step(s):
        s["out"] = yt.paged_attention(q, kn, vn, s["kp"][0], s["vp"][0], s["table"], s["len"])
        s["out2"], s["sel"] = yt.paged_sparse_attention(q, kn, vn, s["kp"][0], s["vp"][0], s["sums"][0], s["table"],
                                                        s["len"], 2)
        s["old"].copy_(s["len"])
        yt.cache_grow(s["ref"], s["table"], s["len"], s["n"], page)
        yt.cache_append(kn[None], vn[None], s["kp"], s["vp"], s["table"], s["old"], n_new=s["n"], key_sums=s["sums"])

    eager, held = fresh(), fresh()
    step(fresh())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(5):
        step(eager)
        torch.randn(1 << 20, device="cuda").sum().item()
        graph.replay()
        torch.cuda.synchronize()
        for name in ("out", "out2", "sel", "ref", "table", "len", "sums"):
            assert torch.equal(held[name], eager[name]), name
        assert torch.equal(held["kp"].view(torch.int16), eager["kp"].view(torch.int16))


def test_two_streams_at_once():
    """Calls on two streams do not share scratch memory."""
    page, d = 16, 128
    g, kp, vp, table, kv_len = cache(2, [5000, 3000], 2, page, d, torch.bfloat16)
    sums = torch.nan_to_num(kp.float()).sum(2)
    work = []
    for i in range(2):
        q, kn, vn = tokens(g, 2, 4, 2, 3, d, torch.bfloat16)
        work.append((q, kn, vn, yt.paged_attention(q, kn, vn, kp, vp, table, kv_len),
                     yt.paged_sparse_attention(q, kn, vn, kp, vp, sums, table, kv_len, 9)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(10):
        got = []
        for s, (q, kn, vn, _, _) in zip(streams, work):
            with torch.cuda.stream(s):
                got.append((yt.paged_attention(q, kn, vn, kp, vp, table, kv_len),
                            yt.paged_sparse_attention(q, kn, vn, kp, vp, sums, table, kv_len, 9)))
        torch.cuda.synchronize()
        for (a, (c, e)), (_, _, _, b, (f, h)) in zip(got, work):
            assert torch.equal(a, b) and torch.equal(c, f) and torch.equal(e, h)
