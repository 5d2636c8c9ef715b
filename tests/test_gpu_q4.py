"""4-bit pages on the GPU: rows into them, their values and attention over them, against q4_ref and window_ref."""
from __future__ import annotations

import math

import pytest
import torch

import q4_ref
import ytensor_amd as yt
from window_ref import Rows, attention, compare

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def kept(k, v, page, d):
    """The pools' values [..., page, d] in float64, as q4_ref reads them."""
    return q4_ref.values(k, page, d, "k"), q4_ref.values(v, page, d, "v")


# ------------------------------------------------------------------ rows into the pages

def odd_rows(g, shape, dt):
    """Random rows of many sizes with zeros, ties, group borders, tiny, huge and missing values."""
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-12, 9, (*shape[:-1], 1), generator=g).float())
    x = x.to(dt).flatten(0, -2)
    n = len(x)
    f = torch.finfo(dt)
    special = [torch.zeros(32), torch.full((32,), 7.0), torch.linspace(-6, 6, 32), torch.arange(32) * 0.25 - 4, torch.full((32,), f.tiny),
               torch.full((32,), f.max), torch.full((32,), -f.max), torch.tensor([math.nan] + [1.0] * 31), torch.tensor([1.0] * 31 + [math.inf]),
               torch.tensor([-0.0, 5.0] * 16), torch.full((32,), f.smallest_normal / 2), torch.tensor([7.0078125] + [3.5] * 31)]
    for i, s in enumerate(special):
        x[(i * 5) % n, 32:64] = s.to(dt)
    return x.reshape(shape)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("T,lens,news,path", [(1, [0], [1], False), (40, [3, 0, 77, 16], [40, 0, 17, 1], False), (16, [5, 31, 64], [4, 1, 6], True)])
def test_append(dtype, d, page, T, lens, news, path):
    dt, L, B, Hkv = DT[dtype], 2, len(lens), 2
    g = torch.Generator().manual_seed(T + d)
    need = [-(-(n + m) // page) for n, m in zip(lens, news)]
    P = sum(need) + 2
    table = torch.full((B, max(need) + 1), -1, dtype=torch.int32)
    perm, at = torch.randperm(P, generator=g).tolist(), 0
    for b in range(B):
        for c in range(need[b]):
            table[b, c], at = perm[at], at + 1
    size = yt.cache_q4_bytes(page, d)
    k, v = (torch.randint(0, 256, (L, P, Hkv, size), generator=g).to(torch.uint8) for _ in range(2))
    kn, vn = odd_rows(g, (L, B, Hkv, T, d), dt), odd_rows(g, (L, B, Hkv, T, d), dt)
    take = torch.stack([torch.randperm(T, generator=g) for _ in range(B)]).int() if path else None
    if path:
        take[0, 1], take[2, 0] = -1, T  # rows of zeros
    for ways in range(3):
        kc, vc = k.cuda(), v.cuda()
        status = ints([0])
        kw = [dict(n_new=ints(news)), dict(new_len=ints([n + m for n, m in zip(lens, news)]), status=status),
              dict(n_new=ints(news))][ways]
        knc, vnc = kn.cuda(), vn.cuda()
        if ways == 2:  # rows at other strides, alike for both and not
            knc, vnc = (t.permute(3, 0, 2, 1, 4).contiguous().permute(1, 3, 2, 0, 4) for t in (knc, vnc))
            vnc = vnc.contiguous() if T > 1 else vnc
        yt.cache_append_q4(knc, vnc, kc, vc, table.cuda(), ints(lens), page, path=None if take is None else take.cuda(), **kw)
        assert status.item() == 0
        for pool, new, was, which in ((kc.cpu(), kn, k, "k"), (vc.cpu(), vn, v, "v")):
            want, care = was.clone(), torch.ones(was.shape, dtype=torch.bool)
            for b in range(B):
                for i in range(news[b]):
                    j = i if take is None else int(take[b, i])
                    r = lens[b] + i
                    p = int(table[b, r // page])
                    for l in range(L):
                        for h in range(Hkv):
                            x = new[l, b, h, j:j + 1] if 0 <= j < T else torch.zeros(1, d, dtype=dt)
                            codes, scales = q4_ref.rows(x)
                            q4_ref.put(want[l, p, h], r % page, codes[0], scales[0], page, d, which)
                            for s in torch.nonzero(scales[0] == 255).flatten().tolist():
                                for ch in range(32 * s, 32 * s + 32):
                                    care[l, p, h, q4_ref.place(page, d, r % page, ch, which)[0]] = False
            assert torch.equal(pool[care], want[care])


@pytest.mark.parametrize("d,page", [(64, 16), (128, 32)])
def test_append_to_lengths_that_cannot_be(d, page):
    """What ythip_cache_append_to says of refused sequences, bad lengths and page ids, and rows past those given."""
    L, B, Hkv, T, P = 1, 6, 1, 4, 9
    size = yt.cache_q4_bytes(page, d)
    kn = torch.randn(L, B, Hkv, T, d, device="cuda")
    table = ints([[0, 1], [2, 3], [4, -1], [5, 99], [6, 7], [8, 8]])
    lens = [3, 5, page - 2, page - 1, -1, 2 * page - 1]
    new = [3, 4, page + 2, page + 1, 2, 2 * page + 1]  # none, shorter, onto no page, onto a bad page, from below 0, past the table
    k, v = (torch.full((L, P, Hkv, size), 255, dtype=torch.uint8, device="cuda") for _ in range(2))
    status = ints([0])
    yt.cache_append_q4(kn, kn, k, v, table, ints(lens), page, new_len=ints(new), status=status)
    assert status.item() == yt.CACHE_ERR_INDEX
    touched = sorted(set(torch.nonzero((k != 255).any(-1).any(-1))[:, 1].tolist()))
    assert touched == [4, 5, 8]
    assert (k[0, 4, 0].cpu() == 255).sum() > 0
    # more rows in use than given: zeros, and the bit
    k.fill_(255), v.fill_(255), status.zero_()
    yt.cache_append_q4(kn[:, :1], kn[:, :1], k, v, ints([[0, 1]]), ints([2]), page, new_len=ints([page + 3]), status=status)
    assert status.item() == yt.CACHE_ERR_INDEX
    kv = q4_ref.values(k[0, :2, 0], page, d, "k")
    vv = q4_ref.values(v[0, :2, 0], page, d, "v")
    for x in (kv, vv):
        assert (x[0, 2:6] != 0).any(-1).all() and (x[0, 6:] == 0).all() and (x[1, :3] == 0).all() and x[0, :2].isnan().all() and x[1, 3:].isnan().all()


def test_append_refuses():
    page, d = 16, 64
    k = torch.zeros(2, 3, 2, yt.cache_q4_bytes(page, d), dtype=torch.uint8, device="cuda")
    kn = torch.zeros(2, 1, 2, 4, d, device="cuda")
    ok = dict(table=ints([[0, 1]]), kv_len=ints([0]), page=page)
    yt.cache_append_q4(kn, kn, k, k.clone(), **ok)
    for bad in (dict(n_new=ints([1]), new_len=ints([1])), dict(status=ints([0]))):
        with pytest.raises(ValueError):
            yt.cache_append_q4(kn, kn, k, k.clone(), **ok, **bad)
    for a in ((kn, kn.half(), k, k.clone()), (kn, kn, k[:1], k[:1]), (kn, kn, k, k.float()), (kn, kn, k[..., :100], k[..., :100]), (kn[0], kn[0], k, k)):
        with pytest.raises(ValueError):
            yt.cache_append_q4(*a, **ok)


# ----------------------------------------------------------------------- values

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (128, 64), (64, 128)])
def test_unpack(dtype, d, page):
    g = torch.Generator().manual_seed(page)
    size = yt.cache_q4_bytes(page, d)
    wide = torch.randint(0, 256, (3, 4, 2, size + 32), generator=g).to(torch.uint8).cuda()
    wide[..., page * d // 2:] = wide[..., page * d // 2:] % 40 + 108
    wide[1, 2, 0, size - 4] = 255
    k, v = wide[::2, :, :, :size], wide[::2, :, :, :size].clone()
    v = wide.clone()[::2, :, :, :size]
    k_out, v_out = yt.cache_unpack_q4(k, v, page, DT[dtype])
    for got, want in zip((k_out, v_out), kept(k, v, page, d)):
        assert torch.equal(got.cpu().double().nan_to_num(9e9), want.to(DT[dtype]).double().nan_to_num(9e9))
    one = yt.cache_unpack_q4(wide[1:2, :, :, :size].contiguous(), wide[1:2, :, :, :size].contiguous(), page, DT[dtype], out=(k_out[:1], v_out[:1]))
    want = kept(wide[1:2, :, :, :size], wide[1:2, :, :, :size], page, d)
    for got, w in zip(one, want):
        assert torch.equal(got.isnan().cpu(), w.isnan()) and w.isnan().sum() == 32
        assert torch.equal(got.cpu().double().nan_to_num(9e9), w.to(DT[dtype]).double().nan_to_num(9e9))
    with pytest.raises(ValueError):
        yt.cache_unpack_q4(k, v, page, DT[dtype], out=(k_out, v_out[:1]))
    with pytest.raises(ValueError):
        yt.cache_unpack_q4(k, v, page * 4, DT[dtype])
    with pytest.raises(ValueError):
        yt.cache_unpack_q4(k, v.contiguous(), page, DT[dtype])


# -------------------------------------------------------------------- attention

def cache4(seed, lens, Hkv, page, d, dt, spare=3):
    """4-bit pools of random rows and a table of scattered pages; rows that no sequence uses hold codes at random and
    scales of NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    P = sum(need) + spare
    perm = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), max(max(need), 1) + 1), -7, dtype=torch.int32)
    used, at = torch.zeros(P, page, dtype=torch.bool), 0
    for b, n in enumerate(lens):
        for c in range(need[b]):
            table[b, c] = perm[at]
            used[perm[at], :min(page, n - c * page)] = True
            at += 1
    pools = []
    for which in "kv":
        x = torch.randn(P, Hkv, page, d, generator=g) * torch.exp2(torch.randint(-2, 2, (P, Hkv, page, 1), generator=g).float())
        blocks = q4_ref.pack(x.to(dt), which)
        scale = q4_ref.maps(page, d, which)[2][:, ::32]  # [page, groups]
        for p in range(P):
            if not used[p].all():
                blocks[p][:, scale[~used[p]].flatten()] = 255
        pools.append(blocks.cuda())
    return g, *pools, table.cuda(), ints(lens)


def tokens(g, B, Hq, Hkv, T, d, dt):
    return tuple(torch.randn(B, h, T, d, generator=g).to(dt).cuda() for h in (Hq, Hkv, Hkv))


def tree(g, B, T, far=5):
    back = torch.randint(1, far, (B, T), generator=g)
    return torch.clamp(torch.arange(T)[None] - back, min=-1).int().cuda()


def rows4(k, v, table, kv_len, page, d):
    return Rows(*kept(k, v, page, d), table, kv_len)


@pytest.mark.parametrize("lens", [[0], [1], [15, 16, 17], [300], [0, 64, 1000, 1, 33]], ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("T,kind", [(1, "chain"), (2, "tree"), (7, "tree"), (33, "chain"), (65, "tree"), (1, "none")])
@pytest.mark.parametrize("dtype,d,Hkv,G,page", [("bf16", 128, 2, 2, 16), ("f16", 64, 1, 5, 32), ("f32", 128, 2, 1, 64),
                                                 ("bf16", 64, 1, 17, 128), ("f32", 64, 1, 8, 16), ("f16", 128, 1, 4, 16)])
def test_attention(dtype, d, Hkv, G, page, T, kind, lens):
    dt, B, Hq = DT[dtype], len(lens), Hkv * G
    g, k, v, table, kv_len = cache4(len(lens) * 1000 + T, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hq, Hkv, T, d, dt)
    if kind == "none":
        kn = vn = None
    parents = tree(g, B, T) if kind == "tree" else None
    tree_len = ints([max(0, T - b) for b in range(B)]) if B > 1 else None
    out = torch.full((B, Hq, T, d), 7.0, dtype=dt, device="cuda")
    before = out.clone()
    yt.paged_attention_q4(q, kn, vn, k, v, table, kv_len, page, parents=parents, tree_len=tree_len, out=out)
    want, tol = attention(q, kn, vn, rows4(k, v, table, kv_len, page, d), kv_len, parents, tree_len)
    compare(out, want, tol, before)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (7, 1), (40, 17), (64, 64), (100, 4), (333, 0), (5000, 2), (60, 1000)])
@pytest.mark.parametrize("T,kind", [(1, "chain"), (7, "tree"), (33, "tree"), (70, "chain"), (130, "tree"), (3, "none")])
@pytest.mark.parametrize("dtype,d,Hkv,G,page", [("bf16", 128, 2, 2, 16), ("f16", 64, 1, 5, 32), ("f32", 128, 1, 1, 64)])
def test_window(dtype, d, Hkv, G, page, T, kind, window, sinks):
    dt, lens = DT[dtype], [0, 1, 64, 700, 333]
    B = len(lens)
    g, k, v, table, kv_len = cache4(T + window, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    if kind == "none":
        kn = vn = None
    parents = tree(g, B, T) if kind == "tree" else None
    tree_len = ints([max(0, T - b) for b in range(B)])
    out = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
    before = out.clone()
    yt.paged_attention_q4(q, kn, vn, k, v, table, kv_len, page, parents=parents, tree_len=tree_len, out=out, window=window, sinks=sinks)
    want, tol = attention(q, kn, vn, rows4(k, v, table, kv_len, page, d), kv_len, parents, tree_len, window, sinks)
    compare(out, want, tol, before)


@pytest.mark.parametrize("dtype,B,Hkv,G,d,T,n,page,window,sinks", [
    ("bf16", 1, 2, 2, 128, 1, 40000, 64, 0, 0), ("f16", 2, 1, 8, 128, 40, 9000, 16, 0, 0), ("f32", 1, 1, 4, 64, 3, 20001, 1024, 0, 0),
    ("bf16", 1, 1, 16, 64, 130, 5000, 32, 0, 0), ("bf16", 3, 8, 2, 128, 4, 7001, 4096, 0, 0), ("f32", 1, 2, 2, 128, 70, 3001, 32, 0, 0),
    ("f16", 40, 1, 1, 64, 1, 777, 16, 0, 0), ("bf16", 1, 2, 2, 128, 1, 40000, 64, 20000, 5), ("f16", 2, 1, 8, 128, 40, 9000, 16, 3000, 100),
    ("bf16", 1, 1, 16, 64, 130, 5000, 32, 2047, 1), ("f32", 1, 2, 2, 128, 70, 3001, 32, 3000, 33), ("bf16", 150, 1, 1, 64, 1, 300, 16, 0, 0),
    ("bf16", 2, 1, 2, 64, 700, 900, 32, 0, 0), ("f16", 2, 1, 2, 64, 700, 30, 32, 64, 40), ("f32", 1, 1, 2, 64, 300, 0, 16, 100, 5)])
def test_attention_over_long_caches(dtype, B, Hkv, G, d, T, n, page, window, sinks):
    """The split and its merge, many row tiles, ragged batches, the default out and a scale."""
    dt = DT[dtype]
    lens = [max(0, n - (n - 5) * b // max(B - 1, 1)) if B > 1 else n for b in range(B)]
    g, k, v, table, kv_len = cache4(n, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    for parents in (None, tree(g, B, T)):
        for scale in (0.2, -0.1):
            out = yt.paged_attention_q4(q, kn, vn, k, v, table, kv_len, page, parents=parents, scale=scale, window=window, sinks=sinks)
            want, tol = attention(q, kn, vn, rows4(k, v, table, kv_len, page, d), kv_len, parents, None, window, sinks, scale=scale)
            compare(out, want, tol)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("f16", 128), ("f32", 128)])
def test_strides_and_bad_pages(dtype, d):
    """Pools cut out of wider ones, strided queries and outputs, page ids outside the pool (their rows are hidden)."""
    dt, page, Hkv, B, T = DT[dtype], 16, 2, 3, 5
    lens = [100, 47, 260]
    g, k, v, table, kv_len = cache4(1, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, 4, Hkv, T, d, dt)
    table[0, 2], table[0, 3], table[2, 0], table[2, 16], table[1, 2] = -1, len(k), 1 << 30, -5, -(1 << 31)
    wide = [torch.zeros(len(k), 3, 2 * k.shape[-1], dtype=torch.uint8, device="cuda") for _ in range(2)]
    for w, x in zip(wide, (k, v)):
        w[:, :2, :x.shape[-1]] = x
    kw, vw = (w[:, :2, :k.shape[-1]] for w in wide)
    turned = lambda t: t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # noqa: E731
    out = torch.zeros(B, T, 4, d, dtype=dt, device="cuda").permute(0, 2, 1, 3)
    yt.paged_attention_q4(turned(q), turned(kn), vn, kw, vw, table, kv_len, page, out=out)
    want, tol = attention(q, kn, vn, rows4(k, v, table, kv_len, page, d), kv_len)
    compare(out, want, tol)
    assert torch.equal(out, yt.paged_attention_q4(q, kn, vn, k, v, table, kv_len, page))
    for bad in (dict(page=32), dict(k_pool=k.float()), dict(k_pool=k[..., :-16]), dict(k_new=None), dict(v_new=vn.double()), dict(q=q[0])):
        with pytest.raises(ValueError):
            yt.paged_attention_q4(**(dict(q=q, k_new=kn, v_new=vn, k_pool=k, v_pool=v, table=table, kv_len=kv_len, page=page) | bad))


@pytest.mark.parametrize("columns,pages", [(3, 0), (0, 0), (0, 5)])
@pytest.mark.parametrize("page", [16, 128, 8192])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64)])
def test_no_pages_and_no_columns(dtype, d, page, columns, pages):
    """Every cached row is hidden, or there is none: the new tokens alone, and zeros without them."""
    dt, Hkv, G, B = DT[dtype], 2, 4, 2
    g = torch.Generator().manual_seed(page + columns)
    k, v = (torch.full((pages, Hkv, yt.cache_q4_bytes(page, d)), 255, dtype=torch.uint8, device="cuda") for _ in range(2))
    table = torch.randint(-2, 4, (B, columns), generator=g).int().cuda()
    kv_len = ints([2 * page + 9, 5])
    rows = Rows(*(torch.zeros(pages, Hkv, page, d) for _ in range(2)), table, ints([2 * page + 9, 5] if columns else [0, 0]))
    used = kv_len if columns else ints([0, 0])
    for T in (1, 5, 70):
        for window, sinks in ((0, 0), (3, 40)):
            q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
            out = yt.paged_attention_q4(q, kn, vn, k, v, table, kv_len, page, window=window, sinks=sinks)
            want, tol = attention(q, kn, vn, rows, used, None, None, window, sinks)
            compare(out, want, tol)
            assert (yt.paged_attention_q4(q, None, None, k, v, table, kv_len, page, window=window, sinks=sinks) == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T", [1, 9, 40, 140])
@pytest.mark.parametrize("d", [64, 128])
def test_groups_without_a_value(dtype, T, d):
    """A NaN scale in V reaches its 32 channels of the queries that see the row, one in K all of them; under a window
    those that do not see the row are as without it."""
    dt, Hkv, G, page, n, window, sinks = DT[dtype], 1, 2, 16, 200, 50, 2
    g, k, v, table, kv_len = cache4(T, [n], Hkv, page, d, dt)
    q, kn, vn = tokens(g, 1, G, Hkv, T, d, dt)
    clean = rows4(k, v, table, kv_len, page, d)
    last = n + min(T - 1, 3) + 1 - window  # the last token that sees row `last` is min(T - 1, 3)
    def spoil(pool, which, r, grp):
        block = pool[int(table[0, r // page]), 0]
        block[q4_ref.place(page, d, r % page, 32 * grp, which)[2]] = 255
    vb = v.clone()
    spoil(vb, "v", last, 1)
    spoil(vb, "v", 100, 0)
    kb = k.clone()
    spoil(kb, "k", 100, 1)
    out = yt.paged_attention_q4(q, kn, vn, kb, vb, table, kv_len, page, window=window, sinks=sinks)
    want, tol = attention(q, kn, vn, clean, kv_len, None, None, window, sinks)
    hit = out[:, :, :min(T - 1, 3) + 1].cpu()
    assert hit[..., 32:64].isnan().all()
    keep = [i for i in range(d) if not 32 <= i < 64]
    compare(out[..., keep], want[..., keep], tol[..., keep])
    compare(out[:, :, 4:], want[:, :, 4:], tol[:, :, 4:]) if T > 4 else None
    every = yt.paged_attention_q4(q, kn, vn, k, vb, table, kv_len, page).cpu()
    assert every[..., :64].isnan().all() and torch.isfinite(every[..., 64:]).all()
    assert yt.paged_attention_q4(q, kn, vn, kb, v, table, kv_len, page).isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T", [7, 70])
def test_new_tokens_that_are_not_finite(dtype, T):
    """NaN and infinities in K and V of new tokens reach the tokens below them in the tree, and no other."""
    dt, Hkv, G, page, d, n = DT[dtype], 1, 2, 16, 128, 60
    g, k, v, table, kv_len = cache4(T, [n], Hkv, page, d, dt)
    q, kn, vn = tokens(g, 1, G, Hkv, T, d, dt)
    parents = torch.arange(-2, T - 2, dtype=torch.int32)[None].clamp(min=-1).cuda()  # two chains, the odd and the even
    vb, kb = vn.clone(), kn.clone()
    vb[0, 0, 1, 5], vb[0, 0, 3, 100] = math.inf, math.nan
    want, tol = attention(q, kn, vn, rows4(k, v, table, kv_len, page, d), kv_len, parents)
    out = yt.paged_attention_q4(q, kn, vb, k, v, table, kv_len, page, parents=parents)
    compare(out[:, :, ::2], want[:, :, ::2], tol[:, :, ::2])
    assert (out[:, :, 1::2, 5] == math.inf).all() and out[:, :, 3::2, 100].isnan().all() and torch.isfinite(out[:, :, 1, 100]).all()
    kb[0, 0, 1, 7] = math.nan
    out = yt.paged_attention_q4(q, kb, vn, k, v, table, kv_len, page, parents=parents)
    compare(out[:, :, ::2], want[:, :, ::2], tol[:, :, ::2])
    assert out[:, :, 1::2].isnan().all()
    # a key of -inf in one channel: no weight for queries that are positive there
    kb[0, 0, 1, 7] = -math.inf
    q2 = q.clone()
    q2[..., 7] = q2[..., 7].abs() + 0.1
    hidden = kn.clone()
    out = yt.paged_attention_q4(q2, kb, vn, k, v, table, kv_len, page, parents=parents)
    cut = parents.clone()
    cut[0, 3:4] = -1  # token 3 on without token 1
    want, tol = attention(q2, kn, vn, rows4(k, v, table, kv_len, page, d), kv_len, cut)
    rest = [t for t in range(T) if t != 1]
    compare(out[:, :, rest], want[:, :, rest], tol[:, :, rest])


@pytest.mark.parametrize("kind,window,sinks", [("chain", 0, 0), ("tree", 0, 0), ("chain", 70, 0), ("chain", 100, 90), ("tree", 5, 40)])
@pytest.mark.parametrize("dtype,d,G", [("bf16", 128, 1), ("bf16", 64, 3), ("f16", 128, 1), ("f32", 64, 2)])
def test_long_chunks_with_values_that_are_not_finite(dtype, d, G, kind, window, sinks):
    """Infinities and NaN in V of new tokens, in tiles next to each other and apart: NaN or that infinity where a token sees
    one, and within the bound everywhere else."""
    dt, Hkv, page, T, lens = DT[dtype], 1, 16, 330, [37, 0]
    g, k, v, table, kv_len = cache4(T + window, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, 2, Hkv * G, Hkv, T, d, dt)
    parents = tree(g, 2, T, 40) if kind == "tree" else None
    tree_len = ints([T, T - 9])
    bad = vn.clone()
    for b, t, ch, x in ((0, 0, 3, math.inf), (0, 70, 9, -math.inf), (0, 140, 3, -math.inf), (0, 329, d - 1, math.nan), (1, 64, 0, math.nan),
                        (1, 130, 17, math.inf), (1, 131, 40, math.inf), (1, 325, 5, math.nan)):
        bad[b, 0, t, ch] = x
    out = yt.paged_attention_q4(q, kn, bad, k, v, table, kv_len, page, parents=parents, tree_len=tree_len, window=window, sinks=sinks)
    rows = rows4(k, v, table, kv_len, page, d)
    want, _ = attention(q, kn, bad, rows, kv_len, parents, tree_len, window, sinks)
    zeros = torch.where(torch.isfinite(bad), bad, 0.0)
    fine, tol = attention(q, kn, zeros, rows, kv_len, parents, tree_len, window, sinks)
    o = out.cpu().double()
    for b in range(2):
        n = int(tree_len[b])
        w, f, tl, got = want[b, :, :n], fine[b, :, :n], tol[b, :, :n], o[b, :, :n]
        assert torch.equal(w.isnan(), got.isnan()) and torch.equal(w[w.isinf()], got[w.isinf()])
        ok = torch.isfinite(w)
        assert ((got - f).abs()[ok] <= tl[ok]).all()


@pytest.mark.parametrize("dtype", ["f16", "f32", "bf16"])
def test_large_and_close_scores(dtype):
    """Queries whose scores are far from 0 and near each other: the weights keep their order."""
    dt, page, d, n = DT[dtype], 32, 128, 500
    g, k, v, table, kv_len = cache4(2, [n], 1, page, d, dt)
    q, kn, vn = tokens(g, 1, 4, 1, 3, d, dt)
    q = (q.float() * torch.tensor([1e-3, 30.0, 200.0, 1.0], device="cuda")[None, :, None, None]).to(dt)
    want, tol = attention(q, kn, vn, rows4(k, v, table, kv_len, page, d), kv_len)
    compare(yt.paged_attention_q4(q, kn, vn, k, v, table, kv_len, page), want, tol)


@pytest.mark.parametrize("dtype,d", [("f16", 64), ("f32", 128), ("bf16", 128), ("bf16", 64), ("f16", 128), ("f32", 64)])
def test_queries_of_all_sizes(dtype, d):
    """Channels of a query far apart in size, tiny and zero queries; one that is not finite is NaN and no other is."""
    dt, page, n, T = DT[dtype], 16, 150, 5
    g, k, v, table, kv_len = cache4(3, [n], 1, page, d, dt)
    q, kn, vn = tokens(g, 1, 4, 1, T, d, dt)
    size = torch.exp2(torch.randint(-14, 4, q.shape, generator=g).float()).cuda()
    q = (q.float() * size).to(dt)
    q[0, 0, 0], q[0, 1, 1] = 0.0, q[0, 1, 1] * torch.finfo(dt).tiny
    q[0, 2, 2, 32:] = 0.0
    want, tol = attention(q, kn, vn, rows4(k, v, table, kv_len, page, d), kv_len)
    compare(yt.paged_attention_q4(q, kn, vn, k, v, table, kv_len, page), want, tol)
    bad = q.clone()
    bad[0, 3, 4, 7], bad[0, 1, 0, 40], bad[0, 2, 1, d - 1] = math.inf, math.nan, -math.inf
    out = yt.paged_attention_q4(bad, kn, vn, k, v, table, kv_len, page).cpu()
    hit = torch.zeros(1, 4, T, dtype=torch.bool)
    hit[0, 3, 4] = hit[0, 1, 0] = hit[0, 2, 1] = True
    assert out[hit].isnan().all()
    compare(out[~hit], want[~hit], tol[~hit])


# ------------------------------------------------------------------ used together

def test_a_served_step():
    """Two sequences through prompt, drafted steps (attention of a tree, its verification, pages and rows for what is
    kept), a fork, an end and a packed pool: at each step attention over the 4-bit cache equals attention over the
    values of the rows that were kept, and the captured step goes on as the eager one does."""
    dt, Hkv, G, d, page, V, T = torch.bfloat16, 2, 2, 64, 16, 97, 6
    g = torch.Generator().manual_seed(0)
    B, P, columns = 3, 40, 12
    k, v = (torch.zeros(1, P, Hkv, yt.cache_q4_bytes(page, d), dtype=torch.uint8, device="cuda") for _ in range(2))
    ref, table, kv_len = ints([0] * P), ints([[-1] * columns] * B), ints([0] * B)
    status = ints([0])
    held = [torch.zeros(2, Hkv, 0, d, dtype=dt) for _ in range(B)]  # the rows as they came, [K and V]
    old = torch.empty_like(kv_len)

    def grow_and_append(kn, vn, n_new, path=None):
        old.copy_(kv_len)
        yt.cache_grow(ref, table, kv_len, n_new, page, status=status)
        yt.cache_append_q4(kn, vn, k, v, table, old, page, path=path, new_len=kv_len, status=status)

    def keep(kn, vn, counts, path=None):
        for b, m in enumerate(counts):
            at = list(range(m)) if path is None else path[b][:m]
            held[b] = torch.cat([held[b], torch.stack([kn[0, b].cpu()[:, at], vn[0, b].cpu()[:, at]])], 2)

    def check_cache():
        kv, vv = kept(k[0], v[0], page, d)
        for b in range(B):
            n = held[b].shape[2]
            assert kv_len[b].item() == n
            at = table[b].cpu().tolist()
            for got, rows in ((kv, held[b][0]), (vv, held[b][1])):
                mine = torch.cat([got[p] for p in at[:-(-n // page)]], 1)[:, :n] if n else torch.zeros(Hkv, 0, d)
                codes, scales = zip(*(q4_ref.rows(rows[h]) for h in range(Hkv))) if n else ((), ())
                for h in range(Hkv if n else 0):
                    block = torch.zeros(-(-n // 16) * 16 * (d // 2 + d // 32), dtype=torch.uint8)
                    for r in range(n):
                        q4_ref.put(block, r, codes[h][r], scales[h][r], -(-n // 16) * 16, d, "k")
                    assert torch.equal(mine[h], q4_ref.values(block, -(-n // 16) * 16, d, "k")[:n])

    prompt = [30, 17, 0]
    kn, vn = (torch.randn(1, B, Hkv, 30, d, generator=g).to(dt).cuda() for _ in range(2))
    grow_and_append(kn, vn, ints(prompt))
    keep(kn, vn, prompt)
    check_cache()

    q, k1, v1 = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    parents, tree_len = tree(g, B, T, 3), ints([T, T - 1, 0])
    parents[:, 1:].clamp_(min=0)
    head = torch.randn(Hkv * G * d, V, generator=g).to(dt).cuda()
    toks, u, un = ints([[0] * T] * B), torch.zeros(B, T, device="cuda"), torch.zeros(B, device="cuda")
    out = torch.zeros_like(q)
    picks = (ints([[0] * T] * B), ints([0] * B), ints([0] * B))

    def step():
        yt.paged_attention_q4(q, k1, v1, k[0], v[0], table, kv_len, page, parents=parents, tree_len=tree_len, window=20, sinks=4, out=out)
        logits = yt.matmul(out.transpose(1, 2).reshape(B * T, -1), head).view(B, T, V)
        yt.verify_drafts(yt.token_probs(logits, 0.5), toks, u, un, parents=parents, tree_len=tree_len, out=picks)
        grow_and_append(k1[None], v1[None], picks[1], path=picks[0])

    def again(run):
        for t in (q, k1, v1):
            t.copy_(torch.randn(t.shape, generator=g))
        toks.copy_(torch.randint(0, V, (B, T), generator=g))
        u.copy_(torch.rand(B, T, generator=g) * 0.02)
        un.copy_(torch.rand(B, generator=g))
        want, tol = attention(q, k1, v1, rows4(k[0], v[0], table, kv_len, page, d), kv_len, parents, tree_len, 20, 4)
        before = out.clone()
        run()
        torch.cuda.synchronize()
        compare(out, want, tol, before)
        keep(k1[None], v1[None], picks[1].tolist(), picks[0].tolist())
        check_cache()
        assert status.item() == 0 and picks[2][2].item() == -1

    again(step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    keep_state = [t.clone() for t in (ref, table, kv_len, k, v)]
    with torch.cuda.graph(graph):
        step()
    for t, was in zip((ref, table, kv_len, k, v), keep_state):
        assert torch.equal(t, was)  # a capture runs nothing
    for i in range(4):
        again(graph.replay if i % 2 == 0 else step)
    # sequence 2 becomes a copy of 0, 1 ends, the pool is packed
    yt.cache_fork((k, v), ref, table, kv_len, ints([0]), ints([2]), page, status=status)
    held[2] = held[0]
    check_cache()
    yt.cache_free(ref, table, kv_len, ints([1]), page, status=status)
    held[1] = torch.zeros(2, Hkv, 0, d, dtype=dt)
    _, _, live = yt.cache_compact((k, v), ref, table, kv_len, page)
    check_cache()
    assert status.item() == 0 and live.item() == int((ref > 0).sum()) and int(table[0, 0]) < live.item()


def test_two_streams_at_once():
    """Calls on two streams that overlap, each with a workspace of its own, over one pool: what each gives alone, bit for bit,
    in eager calls and as two graphs."""
    cases = []
    for dtype, T, Hkv, G, window in (("bf16", 1, 2, 2, 0), ("bf16", 300, 1, 2, 0), ("f16", 25, 2, 5, 700), ("f32", 40, 1, 4, 0)):
        dt, page, d = DT[dtype], 32, 128
        g, k, v, table, kv_len = cache4(T, [4000, 1777], Hkv, page, d, dt)
        q, kn, vn = tokens(g, 2, Hkv * G, Hkv, T, d, dt)
        want = yt.paged_attention_q4(q, kn, vn, k, v, table, kv_len, page, window=window, sinks=4)
        need = yt.paged_q4_workspace_bytes(dt, 2, Hkv * G, Hkv, T, d, table.shape[1], page, window, 4)
        cases.append((want, [(torch.empty_like(want), torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")) for _ in range(2)],
                      lambda out, ws, a=(q, kn, vn, k, v, table, kv_len, page), w=window: yt.paged_attention_q4(*a, window=w, sinks=4, out=out, workspace=ws)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            for _, to, call in cases:
                call(*to[i])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            for _, to, call in cases if i else reversed(cases):
                call(*to[i])
        graphs.append(graph)
    for kind in ("eager", "graphs", "eager", "graphs"):
        for _, to, _ in cases:
            for out, _ in to:
                out.fill_(7.0)
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                if kind == "graphs":
                    graphs[i].replay()
                else:
                    for _, to, call in cases if i else reversed(cases):
                        call(*to[i])
        torch.cuda.synchronize()
        for want, to, _ in cases:
            for out, _ in to:
                assert torch.equal(out, want)
