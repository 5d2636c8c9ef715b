"""Cases by which the operators of the paged KV cache are judged.

Layout: pools [pages, Hkv, page, d] for K and V (a layer; several layers lie in front as
[layers, ...]), key sums [pages, Hkv, d] in float32 (a page's K rows added up), a page table
[B, columns] and the rows in use kv_len [B], both int32, and a count of users per page, int32.

  attend   attention of T new tokens a sequence (one token, a drafted tree, a chunk of a
           prompt) over the paged cache and their own K / V rows
  sparse   the same over top_k pages, chosen for each token and KV head by
           (sum of the group's queries) . (key sum of the page) in 64 bits
  commit   pages for the accepted rows, then the rows of every layer into them
  fork     sequences that share another's whole pages and get a copy of its last, partial one
  compact  sequences freed, then the live pages moved to the front of the pools

With `own` false everything is plain torch in 32 bits (the page scores in 64).
"""
from __future__ import annotations

import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ES = {"f32": 4, "f16": 2, "bf16": 2}


def _cdiv(a, b):
    return -(-a // b)


def listed():
    return [
        # one token of one short conversation: latency alone
        dict(name="attend 1 token, 300 rows", op="attend", dtype="bf16", B=1, Hq=16, Hkv=8, d=128, T=1, ctx=300, page=16, tree=False),
        # a decode step of a ragged batch of 16, the context of the framework's decode benchmark
        dict(name="attend 16 x 1 token, 8192 rows", op="attend", dtype="bf16", B=16, Hq=16, Hkv=8, d=128, T=1, ctx=8192, page=64, tree=False),
        # drafted trees of 25 tokens for a few ragged sequences, a group of 5
        dict(name="attend 5 x tree of 25, 4097 rows", op="attend", dtype="f16", B=5, Hq=40, Hkv=8, d=128, T=25, ctx=4097, page=32, tree=True),
        # a tree of 64 over one very long context
        dict(name="attend tree of 64, 131072 rows", op="attend", dtype="bf16", B=1, Hq=16, Hkv=8, d=128, T=64, ctx=131072, page=64, tree=True),
        # the reference's own type, one query head to a KV head, small heads
        dict(name="attend 3 x tree of 7, fp32 d 64", op="attend", dtype="f32", B=3, Hq=8, Hkv=8, d=64, T=7, ctx=2000, page=128, tree=True),
        # the next 512 tokens of two prompts over what is cached
        dict(name="attend 2 x chunk of 512, 8192 rows", op="attend", dtype="bf16", B=2, Hq=16, Hkv=8, d=128, T=512, ctx=8192, page=64, tree=False),
        # one token over a very long context, 32 of its 2048 pages
        dict(name="sparse 1 token, 32 of 2048 pages", op="sparse", dtype="bf16", B=1, Hq=16, Hkv=8, d=128, T=1, ctx=131071, page=64, top_k=32, tree=False),
        # a batch with short drafts, each token with pages of its own
        dict(name="sparse 16 x tree of 4, 48 pages", op="sparse", dtype="f16", B=16, Hq=16, Hkv=8, d=128, T=4, ctx=32768, page=64, top_k=48, tree=True),
        # after a verification: the accepted rows (1 to 6 of 16) of 28 layers
        dict(name="commit 16 x path of 16 drafted", op="commit", dtype="bf16", L=28, B=16, Hkv=8, d=128, T=16, ctx=1000, page=64, path=True),
        # after a prompt pass: 512 rows of 28 layers
        dict(name="commit prompt of 512", op="commit", dtype="bf16", L=28, B=1, Hkv=8, d=128, T=512, ctx=37, page=64, path=False),
        # eight samples out of one prompt, and of others
        dict(name="fork 8, 28 layers", op="fork", dtype="bf16", L=28, B=16, n=8, Hkv=8, d=128, ctx=1000, page=64),
        # half the sequences end, the pool is packed
        dict(name="compact 2048 pages, 8 layers", op="compact", dtype="bf16", L=8, B=64, Hkv=8, d=128, ctx=2600, page=64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "sparse", "sparse", "commit", "fork", "compact"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    d = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    Hkv, G = rng.choice([(8, 2), (8, 1), (8, 5), (4, 8), (2, 4), (1, 16), (8, 4), (4, 7)])
    c = dict(op=op, dtype=dtype, d=d, page=page, Hkv=Hkv)
    if op == "attend":
        B, T, ctx = _log(rng, 1, 32), _log(rng, 1, 128), _log(rng, 30, 100000)
        while B * ctx * Hkv * d * ES[dtype] > 1 << 28 or B * T * Hkv * G * ctx > 1 << 27:  # below the largest listed
            B, T, ctx = max(1, B // 2), max(1, T * 2 // 3), max(30, ctx * 4 // 5)
        c.update(B=B, Hq=Hkv * G, T=T, ctx=ctx, tree=rng.random() < 0.7)
    elif op == "sparse":
        B, T, ctx, top = _log(rng, 1, 16), _log(rng, 1, 8), _log(rng, 500, 100000), _log(rng, 2, 64)
        while B * ctx * Hkv * d * ES[dtype] > 1 << 28 or B * T * Hkv * top * page * d * ES[dtype] > 1 << 28:
            B, T, ctx, top = max(1, B // 2), max(1, T // 2), max(500, ctx * 4 // 5), max(2, top * 4 // 5)
        c.update(B=B, Hq=Hkv * G, T=T, ctx=ctx, top_k=top, tree=rng.random() < 0.6)
    elif op == "commit":
        L, B, T, ctx = _log(rng, 1, 28), _log(rng, 1, 16), _log(rng, 1, 500), _log(rng, 1, 1500)
        while L * B * (ctx + T) * Hkv * d * ES[dtype] > 1 << 29:
            B, T, ctx = max(1, B // 2), max(1, T * 2 // 3), max(1, ctx * 2 // 3)
        c.update(L=L, B=B, T=T, ctx=ctx, path=rng.random() < 0.6)
    elif op == "fork":
        L, B, ctx = _log(rng, 1, 28), _log(rng, 2, 24), _log(rng, 1, 1500)
        while L * B * (ctx + page) * Hkv * d * ES[dtype] > 1 << 29:
            B, ctx = max(2, B // 2), max(1, ctx * 2 // 3)
        c.update(L=L, B=B, n=rng.randint(1, B), ctx=ctx)
    else:
        L, B, ctx = _log(rng, 1, 8), _log(rng, 2, 64), _log(rng, 20, 2600)
        while L * B * (ctx + page) * Hkv * d * ES[dtype] > 1 << 29:
            B, ctx = max(2, B // 2), max(20, ctx * 2 // 3)
        c.update(L=L, B=B, ctx=ctx)
    return c


# --------------------------------------------------------------------- inputs

def _lens(c):
    """Rows in use, from ctx down to a quarter of it: the same ones for every seed, in another order."""
    B, ctx = c["B"], c["ctx"]
    return [ctx - (3 * ctx // 4) * b // max(B - 1, 1) for b in range(B)]


def _new(c):
    """New tokens of each sequence: all of them, or a few less in a batch."""
    return [max(1, c["T"] - b % 3) for b in range(c["B"])]


def _accepted(c):
    return [1 + (5 * b) % 6 if c["path"] else c["T"] for b in range(c["B"])]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)


def _cache(c, g, h, layers, slack, columns):
    """Pools of random rows, and sequences whose pages lie scattered over them."""
    dt, page, dev = DT[c["dtype"]], c["page"], "cuda"
    lens = torch.tensor(_lens(c))[torch.randperm(c["B"], generator=h)]
    need = -(-lens // page)
    P = int(need.sum()) + slack
    lead = (layers,) if layers else ()
    s = {"k_pool": torch.randn(*lead, P, c["Hkv"], page, c["d"], generator=g, device=dev, dtype=dt),
         "v_pool": torch.randn(*lead, P, c["Hkv"], page, c["d"], generator=g, device=dev, dtype=dt)}
    perm = torch.randperm(P, generator=h)
    table = torch.full((c["B"], columns), -1, dtype=torch.int64)
    cols = torch.arange(columns)[None, :] < need[:, None]
    table[cols] = perm[:int(need.sum())]
    ref = torch.zeros(P, dtype=torch.int32)
    ref[perm[:int(need.sum())]] = 1
    s["table"], s["kv_len"], s["ref"] = table.int().to(dev), lens.int().to(dev), ref.to(dev)
    return s


def _parents(c, h):
    """A drafted tree a sequence: the parent of token t is one of the few before it, or the cache's last row (-1)."""
    t = torch.arange(c["T"])[None, :].expand(c["B"], -1)
    back = torch.randint(1, 6, (c["B"], c["T"]), generator=h)
    return torch.clamp(t - back, min=-1).int()


def prepare(case, seed):
    c, (g, h) = case, _gen(seed)
    dt, dev, page, B = DT[c["dtype"]], "cuda", c["page"], c["B"]
    if c["op"] in ("attend", "sparse"):
        s = _cache(c, g, h, 0, 3, _cdiv(c["ctx"], page) + 2)
        Hq, Hkv, T, d = c["Hq"], c["Hkv"], c["T"], c["d"]
        s["q"] = torch.randn(B, Hq, T, d, generator=g, device=dev, dtype=dt)
        s["k_new"] = torch.randn(B, Hkv, T, d, generator=g, device=dev, dtype=dt)
        s["v_new"] = torch.randn(B, Hkv, T, d, generator=g, device=dev, dtype=dt)
        s["tree_len"] = torch.tensor(_new(c), dtype=torch.int32, device=dev)
        s["parents"] = _parents(c, h).to(dev) if c["tree"] else None
        s["out"] = torch.zeros(B, Hq, T, d, device=dev, dtype=dt)
        if c["op"] == "sparse":
            s["key_sums"] = s["k_pool"].sum(2, dtype=torch.float32)
    elif c["op"] == "commit":
        L, Hkv, T, d = c["L"], c["Hkv"], c["T"], c["d"]
        s = _cache(c, g, h, L, B * (_cdiv(T, page) + 1) + 2, _cdiv(c["ctx"] + T, page) + 1)
        s["key_sums"] = s["k_pool"].sum(3, dtype=torch.float32)
        s["k_new"] = torch.randn(L, B, Hkv, T, d, generator=g, device=dev, dtype=dt)
        s["v_new"] = torch.randn(L, B, Hkv, T, d, generator=g, device=dev, dtype=dt)
        s["n_new"] = torch.tensor([min(n, T) for n in _accepted(c)], dtype=torch.int32, device=dev)
        s["path"] = None
        if c["path"]:  # ascending picks of the drafted tokens, as a path from the root is
            step = torch.clamp(T // s["n_new"].cpu(), min=1)[:, None]
            first = torch.randint(0, 2, (B, 1), generator=h) * (step > 1)
            s["path"] = torch.clamp(torch.arange(T) * step + first, max=T - 1).int().to(dev)
        s["into"] = (torch.empty_like(s["ref"]), torch.empty_like(s["table"]), torch.empty_like(s["kv_len"]))
    elif c["op"] == "fork":
        n = c["n"]
        s = _cache(c, g, h, c["L"], n + 2, _cdiv(c["ctx"], page) + 1)
        s["key_sums"] = s["k_pool"].sum(3, dtype=torch.float32)
        s["table"] = torch.cat([s["table"], torch.full((n, s["table"].shape[1]), -1, dtype=torch.int32, device=dev)])
        s["kv_len"] = torch.cat([s["kv_len"], torch.zeros(n, dtype=torch.int32, device=dev)])
        src = torch.randint(0, B, (n,), generator=h)
        src[: _cdiv(n, 2)] = src[0]  # several out of one
        s["src"], s["dst"] = src.int().to(dev), (B + torch.randperm(n, generator=h)).int().to(dev)
        s["into"] = (torch.empty_like(s["ref"]), torch.empty_like(s["table"]), torch.empty_like(s["kv_len"]))
    else:
        s = _cache(c, g, h, c["L"], 5, _cdiv(c["ctx"], page))
        s["key_sums"] = s["k_pool"].sum(3, dtype=torch.float32)
        s["seqs"] = torch.randperm(B, generator=h)[: _cdiv(B, 2)].int().to(dev)
        # the first two of those that stay share their first page
        two = sorted(set(range(B)) - set(s["seqs"].tolist()))[:2]
        if len(two) == 2:
            s["ref"][s["table"][two[1], 0].long()] -= 1
            s["table"][two[1], 0] = s["table"][two[0], 0]
            s["ref"][s["table"][two[0], 0].long()] += 1
        for name in ("into", "packed"):
            s[name] = (torch.empty_like(s["ref"]), torch.empty_like(s["table"]), torch.empty_like(s["kv_len"]))
    s["case"] = c
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    s, op = state, state["case"]["op"]
    return {"attend": _attend, "sparse": _sparse, "commit": _commit, "fork": _fork, "compact": _compact}[op](s)


def _paths(parents, T):
    """[B, T, T]: u is t or above it."""
    eye = torch.eye(T, device=parents.device)
    reach = eye + (parents.long()[:, :, None] == torch.arange(T, device=parents.device)).float()
    for _ in range(max(1, T - 1).bit_length()):
        reach = torch.clamp(reach @ reach, max=1.0)
    return reach > 0


def _softmax_out(s, q, parts):
    """sum of p V over the parts (K, V, seen), p the softmax over all of them; q [..., rows, d] in float32."""
    scale = 1.0 / math.sqrt(q.shape[-1])
    scores = torch.cat([torch.where(seen, (q @ k.transpose(-1, -2)) * scale, -math.inf) for k, _, seen in parts], -1)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total, out, at = p.sum(-1, keepdim=True), 0.0, 0
    for k, v, _ in parts:
        out = out + p[..., at:at + k.shape[-2]] @ v
        at += k.shape[-2]
    return torch.where(total > 0, out / torch.clamp(total, min=1e-37), torch.zeros_like(out))


def _seen_new(s, c):
    """[B, T, T]: new token u is seen by t."""
    T, t = c["T"], torch.arange(c["T"], device="cuda")
    if s["parents"] is not None:
        seen = _paths(s["parents"], T)
    else:
        seen = (t[None, :] <= t[:, None])[None].expand(c["B"], T, T)
    return seen & (t < s["tree_len"][:, None])[:, None, :]


def _attend(s):
    c = s["case"]
    if own:
        import ytensor_amd as yt
        return yt.paged_attention(s["q"], s["k_new"], s["v_new"], s["k_pool"], s["v_pool"], s["table"], s["kv_len"],
                                  parents=s["parents"], tree_len=s["tree_len"], out=s["out"])
    B, Hq, Hkv, T, d, page = c["B"], c["Hq"], c["Hkv"], c["T"], c["d"], c["page"]
    G, M = Hq // Hkv, s["table"].shape[1]
    at = torch.clamp(s["table"], min=0).long()
    k, v = (s[n][at].transpose(1, 2).reshape(B, Hkv, M * page, d).float() for n in ("k_pool", "v_pool"))
    q = s["q"].float().reshape(B, Hkv, G * T, d)
    rows = torch.arange(M * page, device="cuda") < s["kv_len"][:, None]
    seen = _seen_new(s, c)[:, None, None].expand(B, Hkv, G, T, T).reshape(B, Hkv, G * T, T)
    o = _softmax_out(s, q, [(k, v, rows[:, None, None, :]), (s["k_new"].float(), s["v_new"].float(), seen)])
    real = torch.arange(T, device="cuda") < s["tree_len"][:, None]
    return torch.where(real[:, None, :, None], o.reshape(B, Hq, T, d).to(DT[c["dtype"]]), s["out"])


def _sparse(s):
    c = s["case"]
    if own:
        import ytensor_amd as yt
        return yt.paged_sparse_attention(s["q"], s["k_new"], s["v_new"], s["k_pool"], s["v_pool"], s["key_sums"],
                                         s["table"], s["kv_len"], c["top_k"], parents=s["parents"],
                                         tree_len=s["tree_len"], out=s["out"])
    B, Hq, Hkv, T, d, page, top = c["B"], c["Hq"], c["Hkv"], c["T"], c["d"], c["page"], c["top_k"]
    G, M, dev = Hq // Hkv, s["table"].shape[1], "cuda"
    table = torch.clamp(s["table"], min=0).long()
    pages = -(-s["kv_len"].long() // page)
    col = torch.arange(M, device=dev)
    q = s["q"].double().reshape(B, Hkv, G, T, d).sum(2)
    score = q @ s["key_sums"][table].double().permute(0, 2, 3, 1).contiguous()
    score = torch.where(col == (pages - 1)[:, None, None, None], math.inf, score)
    score = torch.where(col < pages[:, None, None, None], score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    order = torch.where(order < pages[:, None, None, None], order, M).sort(-1).values
    if M < top:
        order = torch.cat([order, torch.full((B, Hkv, T, top - M), M, device=dev)], -1)
    real = torch.arange(T, device=dev) < s["tree_len"][:, None]
    chosen = order < M
    at = torch.gather(table[:, None, None, :].expand(B, Hkv, T, M), -1, torch.clamp(order, max=M - 1))
    head = torch.arange(Hkv, device=dev)[None, :, None, None]
    k, v = (s[n][at, head].reshape(B, Hkv, T, top * page, d).float() for n in ("k_pool", "v_pool"))
    rows = (order[..., None] * page + torch.arange(page, device=dev)) < s["kv_len"].long()[:, None, None, None, None]
    rows = (rows & chosen[..., None]).reshape(B, Hkv, T, 1, top * page)
    seen = _seen_new(s, c)[:, None, :, None, :].expand(B, Hkv, T, G, T)
    kn, vn = (s[n].float()[:, :, None].expand(B, Hkv, T, T, d) for n in ("k_new", "v_new"))
    qr = s["q"].float().reshape(B, Hkv, G, T, d).transpose(2, 3)
    o = _softmax_out(s, qr, [(k, v, rows), (kn, vn, seen)]).transpose(2, 3).reshape(B, Hq, T, d)
    out = torch.where(real[:, None, :, None], o.to(DT[c["dtype"]]), s["out"])
    sel = torch.where(chosen & real[:, None, :, None], order, -1).int()
    return out, sel


def _free_pages(ref):
    """The pages without a user, lowest first (the others behind them)."""
    return torch.sort((ref > 0).int(), stable=True).indices


def _commit(s):
    c = s["case"]
    if own:
        import ytensor_amd as yt
        ref, table, new_len = yt.cache_grow(s["ref"], s["table"], s["kv_len"], s["n_new"], c["page"], out=s["into"])
        yt.cache_append(s["k_new"], s["v_new"], s["k_pool"], s["v_pool"], table, s["kv_len"], n_new=s["n_new"],
                        path=s["path"], key_sums=s["key_sums"])
        return ref, table, new_len, s["k_pool"], s["v_pool"], s["key_sums"]
    B, T, page, dev = c["B"], c["T"], c["page"], "cuda"
    old, n = s["kv_len"].long(), s["n_new"].long()
    new = old + n
    have, want = -(-old // page), -(-new // page)
    before = torch.cumsum(want - have, 0) - (want - have)
    col = torch.arange(s["table"].shape[1], device=dev)
    fresh = (col >= have[:, None]) & (col < want[:, None])
    page_of = _free_pages(s["ref"])[torch.where(fresh, before[:, None] + col - have[:, None], 0)]
    table = torch.where(fresh, page_of, s["table"].long())
    ref = s["ref"].clone()
    ref[page_of[fresh]] = 1
    i = torch.arange(T, device=dev)
    take = s["path"].long() if s["path"] is not None else i[None, :].expand(B, T)
    b, j = torch.nonzero(i < n[:, None], as_tuple=True)
    pos = old[b] + j
    p = table[b, pos // page]
    for pool, rows in (("k_pool", "k_new"), ("v_pool", "v_new")):
        s[pool][:, p, :, pos % page] = s[rows][:, b, :, take[b, j]]
    bt, slot = torch.nonzero((col >= (old // page)[:, None]) & (col < want[:, None]) & (n > 0)[:, None], as_tuple=True)
    used = torch.arange(page, device=dev) < (new[bt] - slot * page)[:, None]
    touched = table[bt, slot]
    s["key_sums"][:, touched] = torch.where(used[None, :, None, :, None], s["k_pool"][:, touched].float(), 0.0).sum(3)
    return ref, table.int(), new.int(), s["k_pool"], s["v_pool"], s["key_sums"]


def _fork(s):
    c = s["case"]
    if own:
        import ytensor_amd as yt
        ref, table, kv_len = yt.cache_fork((s["k_pool"], s["v_pool"], s["key_sums"]), s["ref"], s["table"], s["kv_len"],
                                           s["src"], s["dst"], c["page"], out=s["into"])
        return ref, table, kv_len, s["k_pool"], s["v_pool"], s["key_sums"]
    page, src, dst = c["page"], s["src"].long(), s["dst"].long()
    n = s["kv_len"][src].long()
    whole, part = n // page, n % page > 0
    fresh = _free_pages(s["ref"])[torch.cumsum(part.long(), 0) - 1]
    rows = s["table"][src].long()
    col = torch.arange(rows.shape[1], device="cuda")
    last = torch.gather(rows, 1, torch.clamp(whole, max=rows.shape[1] - 1)[:, None])[:, 0]
    rows_new = torch.where(col < whole[:, None], rows, torch.where((col == whole[:, None]) & part[:, None], fresh[:, None], s["table"][dst].long()))
    table = s["table"].clone()
    table[dst] = rows_new.int()
    ref = s["ref"].clone()
    shared = rows[col < whole[:, None]]
    ref.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    ref[fresh[part]] = 1
    kv_len = s["kv_len"].clone()
    kv_len[dst] = n.int()
    for pool in ("k_pool", "v_pool", "key_sums"):
        s[pool][:, fresh[part]] = s[pool][:, last[part]]
    return ref, table, kv_len, s["k_pool"], s["v_pool"], s["key_sums"]


def _compact(s):
    c = s["case"]
    if own:
        import ytensor_amd as yt
        ref, table, kv_len = yt.cache_free(s["ref"], s["table"], s["kv_len"], s["seqs"], c["page"], out=s["into"])
        ref, table, live = yt.cache_compact((s["k_pool"], s["v_pool"], s["key_sums"]), ref, table, kv_len, c["page"],
                                            out=s["packed"][:2])
        return ref, table, kv_len, live, s["k_pool"], s["v_pool"], s["key_sums"]
    page, seqs = c["page"], s["seqs"].long()
    col = torch.arange(s["table"].shape[1], device="cuda")
    gone = s["table"][seqs].long()[col < -(-s["kv_len"][seqs] // page)[:, None]]
    ref = s["ref"].clone()
    ref.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    table, kv_len = s["table"].clone(), s["kv_len"].clone()
    table[seqs], kv_len[seqs] = -1, 0
    used = ref > 0
    live = used.sum()
    at = torch.arange(ref.shape[0], device="cuda")
    src, dst = at[used & (at >= live)], at[~used & (at < live)]
    for pool in ("k_pool", "v_pool", "key_sums"):
        s[pool][:, dst] = s[pool][:, src]
    to = at.clone()
    to[src] = dst
    mine = col < -(-kv_len // page)[:, None]
    table = torch.where(mine, to[torch.clamp(table, min=0).long()].int(), table)
    ref[dst], ref[src] = ref[src], 0
    return ref, table, kv_len, live.int().reshape(1), s["k_pool"], s["v_pool"], s["key_sums"]


# ------------------------------------------------------------- work and exact

def work(case):
    c = case
    es, d, page = ES[c["dtype"]], c["d"], c["page"]
    lens = _lens(c)
    row = c["Hkv"] * d * es  # one token's K (or V)
    whole = c["Hkv"] * page * d * es
    if c["op"] == "attend":
        T, B, Hq = c["T"], c["B"], c["Hq"]
        io = B * T * (2 * Hq * d * es + 2 * row)
        return {"bytes": sum(lens) * 2 * row + io + 4 * sum(_cdiv(n, page) for n in lens),
                "flops": sum(4 * Hq * d * t * (n + (t + 1) / 2) for n, t in zip(lens, _new(c)))}
    if c["op"] == "sparse":
        T, B, Hq, Hkv = c["T"], c["B"], c["Hq"], c["Hkv"]
        pages = [_cdiv(n, page) for n in lens]
        picked = [min(c["top_k"], p) for p in pages]
        rows = [t * (k * page - page // 2) for k, t in zip(picked, _new(c))]
        # pages that several tokens choose need reading once; how many those are depends on the data, so they count once a token
        return {"bytes": sum(pages) * Hkv * d * 4 + sum(min(r, n) for r, n in zip(rows, lens)) * 2 * row + B * T * (2 * Hq * d * es + 2 * row),
                "flops": sum(4 * Hq * d * r for r in rows) + sum(2 * Hkv * d * t * p for t, p in zip(_new(c), pages))}
    if c["op"] == "commit":
        rows = sum(min(n, c["T"]) for n in _accepted(c))
        touched = sum(_cdiv(n % page + min(a, c["T"]), page) for n, a in zip(lens, _accepted(c)))
        return {"bytes": c["L"] * (rows * 4 * row + touched * c["Hkv"] * d * 8), "flops": c["L"] * rows * c["Hkv"] * d}
    sums = c["Hkv"] * d * 4
    if c["op"] == "fork":
        return {"bytes": c["n"] * c["L"] * 2 * (2 * whole + sums) + 8 * c["n"] * _cdiv(c["ctx"], page), "flops": 0}
    total = sum(_cdiv(n, page) for n in lens)
    return {"bytes": (total // 4) * c["L"] * 2 * (2 * whole + sums) + 12 * total, "flops": 0}  # about half live, half of those above the middle


def _above(parents, t):
    path = [t]
    while 0 <= parents[path[-1]] < path[-1]:
        path.append(parents[path[-1]])
    return path


def exact(case, seed):
    """The attention sequence by sequence and the key sums page by page, in 64 bits; nothing for what is moved."""
    c = case
    if c["op"] in ("fork", "compact"):
        return None
    s = prepare(c, seed)
    page = c["page"]
    lens, table = s["kv_len"].tolist(), s["table"].tolist()
    if c["op"] == "commit":
        sums, free = s["key_sums"].double(), [p for p, r in enumerate(s["ref"].tolist()) if r == 0]
        for b, (n, more) in enumerate(zip(lens, s["n_new"].tolist())):
            row = table[b][: _cdiv(n, page)]
            while len(row) * page < n + more:
                row.append(free.pop(0))
            for slot in range(n // page, len(row)):
                lo, hi = slot * page, min((slot + 1) * page, n + more)
                total = s["k_pool"][:, row[slot], :, : max(0, min(n, hi) - lo)].double().sum(2)
                picks = [(s["path"][b, p - n].item() if s["path"] is not None else p - n) for p in range(max(lo, n), hi)]
                if picks:
                    total = total + s["k_new"][:, b][:, :, picks].double().sum(2)
                    sums[:, row[slot]] = total
        return [None, None, None, None, None, sums]
    G, scale = c["Hq"] // c["Hkv"], 1.0 / math.sqrt(c["d"])
    out = s["out"].double()
    for b, (n, t_n) in enumerate(zip(lens, s["tree_len"].tolist())):
        parents = s["parents"][b].tolist() if s["parents"] is not None else [t - 1 for t in range(c["T"])]
        pages = torch.tensor(table[b][: _cdiv(n, page)], device="cuda")
        if c["op"] == "attend":
            mask = torch.zeros(t_n, t_n, dtype=torch.bool)
            for t in range(t_n):
                mask[t, _above(parents, t)] = True
            bias = torch.where(mask, 0.0, -math.inf).double().cuda()
            for h in range(c["Hkv"]):
                kc, vc = (torch.cat([s[a][pages, h].reshape(-1, c["d"])[:n], s[m][b, h, :t_n]]).double() for a, m in (("k_pool", "k_new"), ("v_pool", "v_new")))
                for g in range(G):
                    w = scale * (s["q"][b, h * G + g, :t_n].double() @ kc.T)
                    w[:, n:] += bias
                    out[b, h * G + g, :t_n] = torch.softmax(w, -1) @ vc
            continue
        for h in range(c["Hkv"]):
            for t in range(t_n):
                qs = s["q"][b, h * G:(h + 1) * G, t].double()
                rank = (s["key_sums"][pages, h].double() * qs.sum(0)).sum(-1)
                rank[-1] = math.inf
                at = torch.sort(torch.sort(rank, descending=True, stable=True).indices[: c["top_k"]]).values
                rows = (at[:, None] * page + torch.arange(page, device="cuda")).reshape(-1) < n
                path = _above(parents, t)
                kc, vc = (torch.cat([s[a][pages[at], h].reshape(-1, c["d"])[rows], s[m][b, h][path]]).double() for a, m in (("k_pool", "k_new"), ("v_pool", "v_new")))
                out[b, h * G:(h + 1) * G, t] = torch.softmax(scale * (qs @ kc.T), -1) @ vc
    return out if c["op"] == "attend" else [out, None]
