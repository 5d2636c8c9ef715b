"""Attention of new tokens over cached rows in 64 bits, with a window and sinks: what include/ythip.h says of
ythip_paged_attn_window and ythip_paged_attn_q4, one sequence and head at a time."""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def above(parents, t):
    """t, the token above it, ..."""
    path = [t]
    while True:
        up = path[-1] - 1 if parents is None else int(parents[path[-1]])
        if not 0 <= up < path[-1]:
            return path
        path.append(up)


def attention(q, k_new, v_new, cached, kv_len, parents=None, tree_len=None, window=0, sinks=0, scale=0.0):
    """(out, tol) in float64 on the CPU; rows behind tree_len are NaN in out. cached(b, h) -> (positions, K, V) of the rows
    that are there, in float64. tol bounds a kernel that rounds the weights and the result to q's type and else works in
    float32:
      result    half a step of |o|
      weights   half a step each, in the product and their sum alike: at most half a step of sum p |v| + |o|
                (float16: one below 2^-24 of the largest may be lost, 2^-25 max |v| a key)
      float32   a score of d products is off by (d + 3) 2^-24 S, S = |scale| sum |q k|, and an exponential by 2^-22 more;
                sums over n keys by n 2^-24: each against sum p |v|, numerator and denominator"""
    B, Hq, T, d = q.shape
    u = HALF_STEP[q.dtype]
    scale = scale or 1.0 / math.sqrt(d)
    f = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    qd, kn, vn = f(q), f(k_new), f(v_new)
    parents = None if parents is None else parents.cpu().tolist()
    tree_len = [T] * B if tree_len is None else tree_len.cpu().tolist()
    kv_len = kv_len.cpu().tolist()
    reach = window if window else 1 << 60
    out = torch.full((B, Hq, T, d), math.nan, dtype=torch.float64)
    tol = torch.zeros((B, Hq, T, d), dtype=torch.float64)
    Hkv = cached.heads
    G = Hq // Hkv
    for b in range(B):
        tn = min(max(tree_len[b], 0), T)
        for h in range(Hkv):
            at, kc, vc = cached(b, h)
            n = max(kv_len[b], 0)
            see = torch.zeros(tn, len(at) + (0 if kn is None else tn), dtype=torch.bool)
            for t in range(tn):
                path = above(None if parents is None else parents[b], t)
                y = n + len(path) - 1
                see[t, :len(at)] = (y - at < reach) | (at < sinks)
                if kn is not None:
                    for i, a in enumerate(path):
                        see[t, len(at) + a] = i < reach or y - i < sinks
            k = kc if kn is None else torch.cat([kc, kn[b, h, :tn]])
            v = vc if vn is None else torch.cat([vc, vn[b, h, :tn]])
            for t in range(tn):
                kt, vt = k[see[t]], v[see[t]]
                rows = slice(h * G, (h + 1) * G)
                if len(kt) == 0:
                    out[b, rows, t] = 0.0
                    continue
                s = scale * (qd[b, rows, t] @ kt.T)
                p = torch.softmax(s, -1)
                o = p @ vt
                out[b, rows, t] = torch.where((s == -math.inf).all(-1, keepdim=True), 0.0, o)
                av = p @ vt.abs()
                S = (abs(scale) * (qd[b, rows, t].abs() @ kt.abs().T)).amax(-1, keepdim=True)
                f32 = 2.0 ** -24 * (2 * (d + 3) * S + 8 + 2 * len(kt))
                # (a weight below 2^-126 of the largest is no normal float32 and may be lost, in the product and in the
                # sum: 2^-126 (|v| + |o|) a key, which counts where the others' V is exactly 0)
                tol[b, rows, t] = 1.01 * (2 * u * o.abs() + u * av + f32 * av) + 2.0 ** -125 * len(kt) * vt.abs().max()
                if q.dtype == torch.float16:
                    tol[b, rows, t] += 2.0 ** -25 * len(kt) * vt.abs().max()
    return out, tol


class Rows:
    """Rows of pools [P, Hkv, page, d] (of values) by a table."""

    def __init__(self, k_pool, v_pool, table, kv_len):
        self.k, self.v = k_pool.detach().cpu().double(), v_pool.detach().cpu().double()
        self.table, self.len = table.cpu().tolist(), kv_len.cpu().tolist()
        self.pages, self.heads, self.page, self.d = self.k.shape

    def __call__(self, b, h):
        n = min(max(self.len[b], 0), len(self.table[b]) * self.page)
        at, ks, vs = [], [], []
        for s in range(-(-n // self.page)):
            p, r = self.table[b][s], min(self.page, n - s * self.page)
            if 0 <= p < self.pages:
                at += range(s * self.page, s * self.page + r)
                ks.append(self.k[p, h, :r])
                vs.append(self.v[p, h, :r])
        empty = torch.zeros(0, self.d, dtype=torch.float64)
        return torch.tensor(at, dtype=torch.int64), torch.cat([empty, *ks]), torch.cat([empty, *vs])


def compare(out, want, tol, before=None):
    """Every row that is computed within its bound; the others as they were."""
    o = out.detach().cpu().double()
    real = ~torch.isnan(want)
    assert torch.isfinite(o[real]).all()
    worst = ((o - want).abs()[real] / tol[real].clamp(min=1e-300)).max().item() if real.any() else 0.0
    print(f"worst error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0
    if before is not None:
        assert torch.equal(out.cpu()[~real], before.cpu()[~real])
