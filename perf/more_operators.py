"""Cases of serving's operators around the paged KV cache: attention over a cache held in 4 bits, attention with a
sliding window and sinks, rows into a 4-bit cache, and the sampling of a drafted step.

Layout: pools [pages, Hkv, page, d] for K and V, a page table [B, columns] and the rows in use kv_len [B], both int32.
A 4-bit pool is uint8 [layers, pages, Hkv, page (d / 2 + d / 32)]: a page and head is a block of codes, then of scales.
Groups of 32 neighbouring channels of a row share a scale 2^e (a byte, e + 127), a value is a sign, and one of 0, 0.5, 1,
1.5, 2, 3, 4, 6 (codes 0 to 7, the sign 8), channel 2 i in the low half of its byte.
  K  codes [page][d / 2], scales [page][d / 32]
  V  codes [page / 8][16][8 rows][d / 32]: entry i holds channels i d / 16 and on; scales [page / 8][d / 32][8 rows]

  attend4  attention of T new tokens a sequence (one, a drafted tree, a chunk of a prompt) over a 4-bit cache and their
           own K / V rows; with a window a token at position y sees what lies at y - window + 1 and on, and below `sinks`
  window   the same over rows of q's type, with a window
  append4  the new tokens' rows of every layer into a 4-bit cache, and the cache's values
  verify   which drafted tokens are kept, from the target's probabilities and given random numbers, and the next token
  probs    softmax(logits / temperature) over the vocabulary

With `own` false everything is plain torch in 32 bits (sums of probabilities in 64).
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
        dict(name="attend4 1 token, 300 rows", op="attend4", dtype="bf16", B=1, Hq=16, Hkv=8, d=128, T=1, ctx=300, page=16, tree=False, window=0, sinks=0),
        # a decode step of a ragged batch of 16, the context of the framework's decode benchmark
        dict(name="attend4 16 x 1 token, 8192 rows", op="attend4", dtype="bf16", B=16, Hq=16, Hkv=8, d=128, T=1, ctx=8192, page=64, tree=False, window=0, sinks=0),
        # drafted trees of 25 tokens for a few ragged sequences, a group of 5, a window over the cache
        dict(name="attend4 5 x tree of 25, 4097 rows, window 2048", op="attend4", dtype="f16", B=5, Hq=40, Hkv=8, d=128, T=25, ctx=4097, page=32, tree=True, window=2048, sinks=4),
        # the next 512 tokens of two prompts over what is cached
        dict(name="attend4 2 x chunk of 512, 8192 rows", op="attend4", dtype="bf16", B=2, Hq=16, Hkv=8, d=128, T=512, ctx=8192, page=64, tree=False, window=0, sinks=0),
        # a decode step of a batch whose layers look back 1024 rows
        dict(name="window 16 x 1 token, 8192 rows, window 1024", op="window", dtype="bf16", B=16, Hq=16, Hkv=8, d=128, T=1, ctx=8192, page=64, tree=False, window=1024, sinks=4),
        # a long chunk of a prompt in such a layer
        dict(name="window chunk of 2048, 2048 rows, window 1024", op="window", dtype="bf16", B=1, Hq=16, Hkv=8, d=128, T=2048, ctx=2048, page=64, tree=False, window=1024, sinks=4),
        # after a verification: the accepted rows (1 to 6 of 16) of four layers, in the reference's own type
        dict(name="append4 16 x path of 16 drafted, fp32", op="append4", dtype="f32", L=4, B=16, Hkv=8, d=128, T=16, ctx=100, page=64, path=True),
        # after a prompt pass: 512 rows of 28 layers
        dict(name="append4 prompt of 512, 28 layers", op="append4", dtype="bf16", L=28, B=1, Hkv=8, d=128, T=512, ctx=37, page=64, path=False),
        # five drafted tokens of one conversation, drawn from a draft model's probabilities
        dict(name="verify chain of 6", op="verify", dtype="f32", B=1, T=6, V=151936, draft=True),
        # drafted trees of a batch
        dict(name="verify 16 x tree of 16", op="verify", dtype="f32", B=16, T=16, V=151936, draft=False),
        # the logits of one token, and of the trees of a batch
        dict(name="probs 1 row", op="probs", dtype="f32", B=1, T=1, V=151936, temperature=0.7),
        dict(name="probs 16 x 16 rows", op="probs", dtype="bf16", B=16, T=16, V=151936, temperature=1.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["attend4", "attend4", "attend4", "window", "window", "append4", "verify", "probs"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("verify", "probs"):
        B, T, V = _log(rng, 1, 64), _log(rng, 1, 32), _log(rng, 1000, 151936)
        while B * T * V > 1 << 25:
            B, T = max(1, B // 2), max(1, T * 2 // 3)
        c = dict(op=op, dtype=dtype, B=B, T=T, V=V)
        c.update(dict(draft=rng.random() < 0.5) if op == "verify" else dict(temperature=rng.choice([0.3, 0.7, 1.0, 1.3])))
        return c
    d = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    Hkv, G = rng.choice([(8, 2), (8, 1), (8, 5), (4, 8), (2, 4), (1, 16), (8, 4), (4, 7)])
    c = dict(op=op, dtype=dtype, d=d, page=page, Hkv=Hkv)
    if op == "append4":
        L, B, T, ctx = _log(rng, 1, 28), _log(rng, 1, 16), _log(rng, 1, 500), _log(rng, 1, 500)
        while L * B * (ctx + T) * Hkv * d > 1 << 24:
            L, B, T, ctx = max(1, L * 3 // 4), max(1, B // 2), max(1, T * 2 // 3), max(1, ctx * 2 // 3)
        c.update(L=L, B=B, T=T, ctx=ctx, path=rng.random() < 0.6)
        return c
    B, T, ctx = _log(rng, 1, 32), _log(rng, 1, 128), _log(rng, 30, 100000)
    while B * ctx * Hkv * d > 1 << 27 or B * T * Hkv * G * ctx > 1 << 27:  # below the largest listed
        B, T, ctx = max(1, B // 2), max(1, T * 2 // 3), max(30, ctx * 4 // 5)
    window = _log(rng, 16, 8192) if op == "window" or rng.random() < 0.3 else 0
    c.update(B=B, Hq=Hkv * G, T=T, ctx=ctx, tree=rng.random() < 0.6, window=window, sinks=rng.choice([0, 1, 4, 16, 100]) if window else 0)
    return c


# ------------------------------------------------------------- values in 4 bits

def _quantise(x, dtype):
    """x [..., d] in float32: codes uint8 [..., d] and the scales' bytes uint8 [..., d / 32].

    The scale is the smallest power of two by which the largest of a group is 7 at most, so that no value is off by more
    than half a step; a scale never takes values beyond the inputs' type or its normal numbers."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = g.abs().amax(-1)
    e = torch.frexp(top).exponent - 3  # top / 2^e in [4, 8)
    e = e + (torch.ldexp(top, -e) > 7).int()
    e = torch.where(top > 0, e, -125).clamp(-125, 13 if dtype == torch.float16 else 125)
    a = torch.ldexp(g.abs(), -e[..., None])
    # halfway to the even code
    code = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = code + 8 * torch.signbit(g).byte()
    return code.reshape(x.shape), (e + 127).byte()


def _nibbles(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _k_block(code, scale):
    """[..., page, d] and [..., page, d / 32] as the block of a page and head."""
    return torch.cat([_nibbles(code).flatten(-2), scale.flatten(-2)], -1)


def _v_block(code, scale):
    page, d = code.shape[-2:]
    lead = code.shape[:-2]
    code = code.reshape(*lead, page // 8, 8, 16, d // 16).transpose(-3, -2)
    scale = scale.reshape(*lead, page // 8, 8, d // 32).transpose(-2, -1)
    return torch.cat([_nibbles(code.contiguous()).flatten(-4), scale.flatten(-3)], -1)


def _blocks(rows, dtype, block):
    """Rows [n, Hkv, page, d] as 4-bit pages, some at a time."""
    return torch.cat([block(*_quantise(part.float(), dtype)) for part in rows.split(max(1, (1 << 24) // rows[0].numel()))])


def _k_codes(blocks, page, d):
    n = page * d // 2
    b = blocks[..., :n].unflatten(-1, (page, d // 2))
    code = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    return code, blocks[..., n:].unflatten(-1, (page, d // 32))


def _v_codes(blocks, page, d):
    n = page * d // 2
    b = blocks[..., :n].unflatten(-1, (page // 8, 16, 8, d // 32))
    code = torch.stack([b & 15, b >> 4], -1).flatten(-2).transpose(-3, -2)
    scale = blocks[..., n:].unflatten(-1, (page // 8, d // 32, 8)).transpose(-2, -1)
    return code.reshape(*blocks.shape[:-1], page, d), scale.reshape(*blocks.shape[:-1], page, d // 32)


def _values(code, scale):
    mag = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=code.device)[(code & 7).long()]
    v = torch.where(code >= 8, -mag, mag).unflatten(-1, (-1, 32))
    return torch.ldexp(v, scale.int()[..., None] - 127).flatten(-2)


# --------------------------------------------------------------------- inputs

def _lens(c):
    """Rows in use, from ctx down to a quarter of it: the same ones for every seed, in another order."""
    B, ctx = c["B"], c["ctx"]
    return [ctx - (3 * ctx // 4) * b // max(B - 1, 1) for b in range(B)]


def _new(c):
    """New tokens of each sequence: all of them, or a few less in a batch."""
    return [max(1, c["T"] - b % 3) for b in range(c["B"])]


def _accepted(c):
    return [min(c["T"], 1 + (5 * b) % 6) if c["path"] else c["T"] for b in range(c["B"])]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed), torch.Generator().manual_seed(seed)


def _parents(c, h):
    """A drafted tree a sequence: the parent of token t is one of the few before it."""
    t = torch.arange(c["T"])[None, :].expand(c["B"], -1)
    back = torch.randint(1, 6, (c["B"], c["T"]), generator=h)
    return torch.clamp(t - back, min=-1).int()


def _table(c, h, grown, columns):
    """Scattered pages for grown[b] rows a sequence, and the pool's pages."""
    need = -(-torch.tensor(grown) // c["page"])
    pages = int(need.sum()) + 3
    table = torch.full((c["B"], columns), -1, dtype=torch.int32)
    cols = torch.arange(columns)[None, :] < need[:, None]
    table[cols] = torch.randperm(pages, generator=h)[:int(need.sum())].int()
    return table, pages


def prepare(case, seed):
    c, (g, h) = case, _gen(seed)
    dt, dev, B = DT[c["dtype"]], "cuda", c["B"]
    if c["op"] in ("attend4", "window"):
        Hq, Hkv, T, d, page = c["Hq"], c["Hkv"], c["T"], c["d"], c["page"]
        lens = torch.tensor(_lens(c))[torch.randperm(B, generator=h)]
        table, pages = _table(c, h, lens.tolist(), _cdiv(c["ctx"], page) + 2)
        s = {"table": table.to(dev), "kv_len": lens.int().to(dev)}
        k, v = (torch.randn(pages, Hkv, page, d, generator=g, device=dev, dtype=dt) for _ in range(2))
        if c["op"] == "attend4":
            k, v = _blocks(k, dt, _k_block), _blocks(v, dt, _v_block)
        s["k_pool"], s["v_pool"] = k, v
        s["q"] = torch.randn(B, Hq, T, d, generator=g, device=dev, dtype=dt)
        s["k_new"] = torch.randn(B, Hkv, T, d, generator=g, device=dev, dtype=dt)
        s["v_new"] = torch.randn(B, Hkv, T, d, generator=g, device=dev, dtype=dt)
        s["tree_len"] = torch.tensor(_new(c), dtype=torch.int32, device=dev)
        s["parents"] = _parents(c, h).to(dev) if c["tree"] else None
        s["out"] = torch.zeros(B, Hq, T, d, device=dev, dtype=dt)
    elif c["op"] == "append4":
        L, Hkv, T, d, page = c["L"], c["Hkv"], c["T"], c["d"], c["page"]
        order = torch.randperm(B, generator=h)
        lens, n_new = torch.tensor(_lens(c))[order], torch.tensor(_accepted(c))[order]
        table, pages = _table(c, h, (lens + n_new).tolist(), _cdiv(c["ctx"] + T, page) + 1)
        s = {"table": table.to(dev), "kv_len": lens.int().to(dev), "new_len": (lens + n_new).int().to(dev)}
        for name, block in (("k_pool", _k_block), ("v_pool", _v_block)):
            s[name] = torch.stack([_blocks(torch.randn(pages, Hkv, page, d, generator=g, device=dev, dtype=dt), dt, block) for _ in range(L)])
        s["k_new"] = torch.randn(L, B, Hkv, T, d, generator=g, device=dev, dtype=dt)
        s["v_new"] = torch.randn(L, B, Hkv, T, d, generator=g, device=dev, dtype=dt)
        s["path"] = None
        if c["path"]:  # ascending picks of the drafted tokens, as a path from the root is
            step = torch.clamp(T // n_new, min=1)[:, None]
            first = torch.randint(0, 2, (B, 1), generator=h) * (step > 1)
            s["path"] = torch.clamp(torch.arange(T) * step + first, max=T - 1).int().to(dev)
        s["values"] = tuple(torch.empty(L, pages, Hkv, page, d, device=dev, dtype=dt) for _ in range(2))
    elif c["op"] == "verify":
        T, V = c["T"], c["V"]
        logits = 3.0 * torch.randn(B, T, V, generator=g, device=dev)
        s = {"target": torch.softmax(logits, -1).to(dt)}
        s["parents"] = None if c["draft"] else torch.clamp(_parents(c, h), min=0).to(dev)
        above = torch.arange(-1, T - 1, device=dev).clamp(min=0).expand(B, T) if c["draft"] else s["parents"].long()
        # a draft model that is near the target; a tree holds draws after each parent
        near = logits + 0.7 * torch.randn(B, T, V, generator=g, device=dev)
        near = torch.softmax(torch.gather(near, 1, above[..., None].expand(B, T, V)), -1)
        s["draft"] = near.to(dt) if c["draft"] else None
        pick = torch.rand(B, T, 1, generator=g, device=dev) * near.sum(-1, keepdim=True)
        s["tokens"] = (torch.cumsum(near.double(), -1) <= pick).sum(-1).clamp(max=V - 1).int()
        s["tree_len"] = torch.tensor(_new(c), dtype=torch.int32, device=dev)
        s["u"] = torch.rand(B, T, generator=g, device=dev)
        s["u_next"] = torch.rand(B, generator=g, device=dev)
    else:
        s = {"logits": (3.0 * torch.randn(B, c["T"], c["V"], generator=g, device=dev)).to(dt)}
    s["case"] = c
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    s, op = state, state["case"]["op"]
    return {"attend4": _attend4, "window": _window, "append4": _append4, "verify": _verify, "probs": _probs}[op](s)


def _paths(parents, T):
    """[B, T, T]: u is t or above it."""
    eye = torch.eye(T, device=parents.device)
    reach = eye + (parents.long()[:, :, None] == torch.arange(T, device=parents.device)).float()
    for _ in range(max(1, T - 1).bit_length()):
        reach = torch.clamp(reach @ reach, max=1.0)
    return reach > 0


def _softmax_out(q, parts):
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


def _attention(s, k, v):
    """k and v [B, Hkv, columns * page, d] in float32."""
    c = s["case"]
    B, Hq, Hkv, T, d = c["B"], c["Hq"], c["Hkv"], c["T"], c["d"]
    G, dev, window, sinks = Hq // Hkv, "cuda", c["window"] or 1 << 40, c["sinks"]
    t = torch.arange(T, device=dev)
    if s["parents"] is not None:
        above = _paths(s["parents"], T)
        depth = above.sum(-1) - 1
    else:
        above = (t[None, :] <= t[:, None])[None].expand(B, T, T)
        depth = t[None].expand(B, T)
    n = s["kv_len"].long()[:, None]
    pos = n + depth  # [B, T]
    row = torch.arange(k.shape[2], device=dev)
    rows = (row < n)[:, None] & ((pos[..., None] - row < window) | (row < sinks))
    new = above & (t < s["tree_len"][:, None])[:, None]
    new = new & ((pos[:, :, None] - pos[:, None] < window) | (pos < sinks)[:, None])
    spread = lambda m: m[:, None, None].expand(B, Hkv, G, T, m.shape[-1]).reshape(B, Hkv, G * T, -1)  # noqa: E731
    q = s["q"].float().reshape(B, Hkv, G * T, d)
    o = _softmax_out(q, [(k, v, spread(rows)), (s["k_new"].float(), s["v_new"].float(), spread(new))])
    real = t < s["tree_len"][:, None]
    return torch.where(real[:, None, :, None], o.reshape(B, Hq, T, d).to(DT[c["dtype"]]), s["out"])


def _attend4(s):
    c = s["case"]
    if own:
        import ytensor_amd as yt
        return yt.paged_attention_q4(s["q"], s["k_new"], s["v_new"], s["k_pool"], s["v_pool"], s["table"], s["kv_len"], c["page"],
                                     parents=s["parents"], tree_len=s["tree_len"], window=c["window"], sinks=c["sinks"], out=s["out"])
    at = torch.clamp(s["table"], min=0).long()
    k = _values(*_k_codes(s["k_pool"][at], c["page"], c["d"]))
    v = _values(*_v_codes(s["v_pool"][at], c["page"], c["d"]))
    return _attention(s, *(x.transpose(1, 2).reshape(c["B"], c["Hkv"], -1, c["d"]) for x in (k, v)))


def _window(s):
    c = s["case"]
    if own:
        import ytensor_amd as yt
        return yt.paged_attention(s["q"], s["k_new"], s["v_new"], s["k_pool"], s["v_pool"], s["table"], s["kv_len"],
                                  parents=s["parents"], tree_len=s["tree_len"], window=c["window"], sinks=c["sinks"], out=s["out"])
    at = torch.clamp(s["table"], min=0).long()
    return _attention(s, *(s[n][at].transpose(1, 2).reshape(c["B"], c["Hkv"], -1, c["d"]).float() for n in ("k_pool", "v_pool")))


def _append4(s):
    c = s["case"]
    dt, page, d, T, dev = DT[c["dtype"]], c["page"], c["d"], c["T"], "cuda"
    if own:
        import ytensor_amd as yt
        yt.cache_append_q4(s["k_new"], s["v_new"], s["k_pool"], s["v_pool"], s["table"], s["kv_len"], page,
                           path=s["path"], new_len=s["new_len"])
        return yt.cache_unpack_q4(s["k_pool"], s["v_pool"], page, dt, out=s["values"])
    n = (s["new_len"] - s["kv_len"]).long()
    i = torch.arange(T, device=dev)
    take = s["path"].long() if s["path"] is not None else i[None, :].expand(c["B"], T)
    b, j = torch.nonzero(i < n[:, None], as_tuple=True)
    pos = s["kv_len"].long()[b] + j
    p, r = s["table"].long()[b, pos // page], pos % page
    code, scale = _k_codes(s["k_pool"], page, d)
    x, e = _quantise(s["k_new"][:, b, :, take[b, j]].float(), dt)
    code, scale = code.clone(), scale.clone()
    code[:, p, :, r], scale[:, p, :, r] = x, e
    s["k_pool"].copy_(_k_block(code, scale))
    k = _values(code, scale).to(dt)
    code, scale = _v_codes(s["v_pool"], page, d)
    x, e = _quantise(s["v_new"][:, b, :, take[b, j]].float(), dt)
    code, scale = code.clone(), scale.clone()
    code[:, p, :, r], scale[:, p, :, r] = x, e
    s["v_pool"].copy_(_v_block(code, scale))
    return k, _values(code, scale).to(dt)


def _verify(s):
    c = s["case"]
    B, T, V, dev = c["B"], c["T"], c["V"], "cuda"
    if own:
        import ytensor_amd as yt
        return yt.verify_drafts(s["target"], s["tokens"], s["u"], s["u_next"], draft=s["draft"], parents=s["parents"], tree_len=s["tree_len"])
    t, tok = torch.arange(T, device=dev), s["tokens"].long()
    real = (t < s["tree_len"][:, None]) & (t > 0)
    up = (t - 1).expand(B, T) if s["parents"] is None else s["parents"].long()
    of = up.clamp(min=0)
    p = s["target"][torch.arange(B, device=dev)[:, None], of, tok].double()
    if s["draft"] is not None:
        q = torch.gather(s["draft"], 2, tok[..., None])[..., 0].double()
        kept = s["u"].double() * q < p
        removed = None
    else:
        # the children of a token share its number: those before t, each of another token, come first
        sibling = (up[:, :, None] == up[:, None]) & real[:, :, None] & real[:, None]
        before = sibling & (t[None, :] < t[:, None])
        twice = (before & (tok[:, :, None] == tok[:, None])).any(-1)
        w = torch.where(twice, 0.0, p)
        low = (before.double() * w[:, None]).sum(-1)
        x = torch.gather(s["u"].double(), 1, of)
        kept = (x >= low) & (x < low + w)
        removed = real
    kept = (kept & real) | (t == 0)
    step = torch.where(t == 0, -1, up)
    on = (_paths(step, T) & ~kept[:, None]).sum(-1) == 0
    on = on & (t < s["tree_len"][:, None])
    n = on.sum(-1)
    path = torch.where(t < n[:, None], torch.sort((~on).int(), stable=True).indices, -1)
    last = torch.gather(path, 1, (n - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
    rest = s["target"][torch.arange(B, device=dev), last].double()
    if s["draft"] is not None:
        more = last + 1 < s["tree_len"]
        q = s["draft"][torch.arange(B, device=dev), (last + 1).clamp(max=T - 1)].double()
        left = torch.where(more[:, None], (rest - q).clamp(min=0), rest)
        rest = torch.where(left.sum(-1, keepdim=True) > 0, left, rest)
    else:
        child = removed & (up == last[:, None])
        gone = torch.zeros(B, V, device=dev).scatter_add_(1, tok, child.float()) > 0
        left = torch.where(gone, 0.0, rest)
        rest = torch.where(left.sum(-1, keepdim=True) > 0, left, rest)
    cum = torch.cumsum(rest, -1)
    at = (cum <= s["u_next"].double()[:, None] * cum[:, -1:]).sum(-1)
    some = (rest > 0).int()
    at = torch.minimum(at, V - 1 - some.flip(-1).argmax(-1))
    nxt = torch.where((n > 0) & (some.sum(-1) > 0), at, -1)
    return path.int(), n.int(), nxt.int()


def _probs(s):
    if own:
        import ytensor_amd as yt
        return yt.token_probs(s["logits"], s["case"]["temperature"])
    x = s["logits"].float() / s["case"]["temperature"]
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True, dtype=torch.float64).float()


# ------------------------------------------------------------- work and exact

def work(case):
    c = case
    es = ES[c["dtype"]]
    if c["op"] == "probs":
        n = c["B"] * c["T"] * c["V"]
        return {"bytes": n * (es + 4), "flops": 4 * n}
    if c["op"] == "verify":
        rows = 2 if c["draft"] else 1  # of the vocabulary: the target's at the last kept token, the draft's behind it
        return {"bytes": c["B"] * (rows * c["V"] * es + c["T"] * (2 * es + 20)), "flops": c["B"] * rows * c["V"]}
    d, page = c["d"], c["page"]
    row4 = c["Hkv"] * (d // 2 + d // 32)  # one token's K (or V) in 4 bits
    row = c["Hkv"] * d * es
    if c["op"] == "append4":
        rows = c["L"] * sum(_accepted(c))
        pages = sum(_cdiv(n + a, page) for n, a in zip(_lens(c), _accepted(c))) + 3
        whole = 2 * c["L"] * pages * page
        return {"bytes": 2 * rows * (row + row4) + whole * (row4 + row), "flops": 8 * rows * c["Hkv"] * d}
    T, B, Hq = c["T"], c["B"], c["Hq"]
    seen = lambda n, y: y if not c["window"] else min(y, c["window"]) + min(c["sinks"], max(y - c["window"], 0))  # noqa: E731
    pairs = sum(seen(n, n + u + 1) for n, t in zip(_lens(c), _new(c)) for u in range(t))
    rows = sum(min(n, seen(n, n + 1)) for n in _lens(c))
    io = B * T * (2 * Hq * d * es + 2 * row)
    return {"bytes": rows * 2 * (row4 if c["op"] == "attend4" else row) + io + 4 * sum(_cdiv(n, page) for n in _lens(c)),
            "flops": 4 * Hq * d * pairs}


def _above(parents, t):
    path = [t]
    while 0 <= parents[path[-1]] < path[-1]:
        path.append(parents[path[-1]])
    return path


STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _four_bits(x, highest):
    """The values of rows x [..., d] held in 4 bits, in 64 bits: the nearest of a group's values, the even code of two."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    unit = 2.0 ** torch.clamp(torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -200) / 7)), -125, highest)
    unit = torch.where((unit * 3.5 >= top) & (unit > 2.0 ** -125), unit / 2, unit)
    unit = torch.where((unit * 7 < top) & (unit < 2.0 ** highest), unit * 2, unit)
    steps = torch.tensor(STEPS, dtype=torch.float64, device=x.device)
    order = [0, 2, 4, 6, 1, 3, 5, 7]  # even codes first: argmin takes the first of two as near
    off = torch.stack([(g.abs() / unit - steps[i]).abs() for i in order], -1)
    near = steps[torch.tensor(order, device=x.device)][off.argmin(-1)]
    return (near * unit * torch.sign(g)).flatten(-2)


def _stored(blocks, c, which):
    """The float64 values [..., page, d] that blocks' bytes stand for."""
    page, d = c["page"], c["d"]
    codes, e = blocks[..., :page * d // 2], blocks[..., page * d // 2:].long()
    r, ch = torch.meshgrid(torch.arange(page, device=blocks.device), torch.arange(d, device=blocks.device), indexing="ij")
    if which == "k":
        at, se = r * (d // 2) + ch // 2, r * (d // 32) + ch // 32
    else:
        per = d // 16
        at = ((r // 8 * 16 + ch // per) * 8 + r % 8) * (d // 32) + ch % per // 2
        se = (r // 8 * (d // 32) + ch // 32) * 8 + r % 8
    code = (codes[..., at].long() >> (4 * (ch % 2))) & 15
    steps = torch.tensor(STEPS + tuple(-x for x in STEPS), dtype=torch.float64, device=blocks.device)
    return steps[code] * 2.0 ** (e[..., se].double() - 127)


def exact(case, seed):
    """Sequence by sequence and page by page, in 64 bits; nothing for whole numbers."""
    c = case
    if c["op"] == "verify":
        return None
    s = prepare(c, seed)
    if c["op"] == "probs":
        return torch.stack([torch.softmax(x.double() / c["temperature"], -1) for x in s["logits"]])
    page, d = c["page"], c["d"]
    lens, table = s["kv_len"].tolist(), s["table"].tolist()
    if c["op"] == "append4":
        highest, out = 13 if c["dtype"] == "f16" else 125, []
        for which in "kv":
            pool, new = s[which + "_pool"], s[which + "_new"]
            L = pool.shape[0]
            values = torch.stack([_stored(pool[layer], c, which) for layer in range(L)])
            for b, (n, m) in enumerate(zip(lens, s["new_len"].tolist())):
                for i in range(n, m):
                    j = i - n if s["path"] is None else s["path"][b, i - n].item()
                    values[:, table[b][i // page], :, i % page] = _four_bits(new[:, b, :, j], highest)
            out.append(values)
        return tuple(out)
    G, scale = c["Hq"] // c["Hkv"], 1.0 / math.sqrt(d)
    window, sinks, out = c["window"] or 1 << 40, c["sinks"], s["out"].double()
    for b, (n, t_n) in enumerate(zip(lens, s["tree_len"].tolist())):
        parents = s["parents"][b].tolist() if s["parents"] is not None else None
        pages = torch.tensor(table[b][: _cdiv(n, page)], device="cuda")
        mask = torch.zeros(t_n, n + t_n, dtype=torch.bool)
        row = torch.arange(n)
        for t in range(t_n):
            path = _above(parents, t) if parents else list(range(t, -1, -1))
            y = n + len(path) - 1
            mask[t, :n] = (y - row < window) | (row < sinks)
            mask[t, [n + u for i, u in enumerate(path) if i < window or y - i < sinks]] = True
        bias = torch.where(mask, 0.0, -math.inf).double().cuda()
        for h in range(c["Hkv"]):
            if c["op"] == "attend4":
                kc, vc = (_stored(s[w + "_pool"][pages, h], c, w).reshape(-1, d)[:n] for w in "kv")
            else:
                kc, vc = (s[w + "_pool"][pages, h].reshape(-1, d)[:n].double() for w in "kv")
            kc, vc = torch.cat([kc, s["k_new"][b, h, :t_n].double()]), torch.cat([vc, s["v_new"][b, h, :t_n].double()])
            for g in range(G):
                w = scale * (s["q"][b, h * G + g, :t_n].double() @ kc.T) + bias
                out[b, h * G + g, :t_n] = torch.softmax(w, -1) @ vc
    return out
