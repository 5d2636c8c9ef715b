"""The paged cache's operators in 64 bits and plain Python, for the tests: what
include/ythip.h says of them, one row and one page at a time."""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def path_of(parents, t):
    """t and what is above it."""
    if parents is None:
        return list(range(t + 1))
    path = [t]
    while 0 <= parents[path[-1]] < path[-1]:
        path.append(int(parents[path[-1]]))
    return sorted(path)


def attention(q, k_new, v_new, k_pool, v_pool, table, kv_len, parents=None, tree_len=None, scale=0.0, sel=None):
    """(out, tol) in float64 on the CPU; rows behind tree_len are NaN in out. tol bounds a kernel that
    rounds the weights p and the result to q's type and else works in float32:
      result      half a step of |o|
      weights     each half a step off, in the product and in their sum alike: sum (w' - w) v / sum w' is
                  sum (w' - w) (v - o) / sum w', at most half a step of sum p |v - o| <= sum p |v| + |o|
                  (and in float16, where a weight below 2^-24 of the largest is lost, 2^-25 max |v| a key)
      float32     a score of d products is off by (d + 3) 2^-24 S, S = scale sum |q k| its largest, and an exponential
                  by 2^-22 more; the sums over n keys by n 2^-24: each against sum p |v|, numerator and denominator
    """
    B, Hq, T, d = q.shape
    P, Hkv, page, _ = k_pool.shape
    G, u = Hq // Hkv, HALF_STEP[q.dtype]
    scale = scale or 1.0 / math.sqrt(d)
    f = lambda t: None if t is None else t.detach().cpu().double()  # noqa: E731
    qd, kn, vn, kp, vp = f(q), f(k_new), f(v_new), f(k_pool), f(v_pool)
    table, kv_len = table.cpu(), kv_len.cpu().tolist()
    parents = None if parents is None else parents.cpu().tolist()
    tree_len = [T] * B if tree_len is None else tree_len.cpu().tolist()
    out = torch.full((B, Hq, T, d), math.nan, dtype=torch.float64)
    tol = torch.zeros((B, Hq, T, d), dtype=torch.float64)
    for b in range(B):
        n = min(max(kv_len[b], 0), table.shape[1] * page)
        for h in range(Hkv):
            def cached(slots):
                ks, vs = [], []
                for s in slots:
                    p, r = int(table[b, s]), min(page, n - s * page)
                    if 0 <= p < P and r > 0:
                        ks.append(kp[p, h, :r])
                        vs.append(vp[p, h, :r])
                return ks, vs
            every = cached(range(-(-n // page))) if sel is None else None
            for t in range(min(max(tree_len[b], 0), T)):
                ks, vs = every if sel is None else cached([int(s) for s in sel[b, h, t] if s >= 0])
                if kn is not None:
                    at = path_of(None if parents is None else parents[b], t)
                    ks, vs = ks + [kn[b, h, at]], vs + [vn[b, h, at]]
                rows = slice(h * G, (h + 1) * G)
                if not ks:
                    out[b, rows, t] = 0.0
                    continue
                k, v = torch.cat(ks), torch.cat(vs)
                s = scale * (qd[b, rows, t] @ k.T)
                p = torch.softmax(s, -1)
                o = p @ v
                out[b, rows, t] = torch.where((s == -math.inf).all(-1, keepdim=True), 0.0, o)
                av = p @ v.abs()
                S = (abs(scale) * (qd[b, rows, t].abs() @ k.abs().T)).amax(-1, keepdim=True)
                f32 = 2.0 ** -24 * (2 * (d + 3) * S + 8 + 2 * len(k))
                tol[b, rows, t] = 1.01 * (2 * u * o.abs() + u * av + f32 * av)
                if q.dtype == torch.float16:
                    tol[b, rows, t] += 2.0 ** -25 * len(k) * v.abs().max()
    return out, tol


def select(q, key_sums, table, kv_len, page, top_k, tree_len=None):
    """The chosen columns [B, Hkv, T, top_k], ascending, then -1."""
    B, Hq, T, d = q.shape
    P, Hkv, _ = key_sums.shape
    G = Hq // Hkv
    qd, ks = q.cpu().double(), key_sums.cpu().double()
    table, kv_len = table.cpu(), kv_len.cpu().tolist()
    tree_len = [T] * B if tree_len is None else tree_len.cpu().tolist()
    sel = torch.full((B, Hkv, T, top_k), -1, dtype=torch.int32)
    for b in range(B):
        n = -(-min(max(kv_len[b], 0), table.shape[1] * page) // page)
        for h in range(Hkv):
            for t in range(min(max(tree_len[b], 0), T)):
                qs = qd[b, h * G:(h + 1) * G, t].sum(0)
                rank = []
                for i in range(n):
                    p = int(table[b, i])
                    s = float((qs * ks[p, h]).sum()) if 0 <= p < P else -math.inf
                    s = -math.inf if math.isnan(s) else s
                    rank.append((0 if i == n - 1 else 1, -s, i))
                at = sorted(i for _, _, i in sorted(rank)[:top_k])
                sel[b, h, t, :len(at)] = torch.tensor(at, dtype=torch.int32)
    return sel


class Pages:
    """The bookkeeping as plain lists; pools are lists of CPU tensors [L, P, ...]."""

    def __init__(self, ref, table, kv_len, page, pools=()):
        self.ref, self.table, self.len = ref.cpu().tolist(), table.cpu().tolist(), kv_len.cpu().tolist()
        self.page, self.pools, self.status = page, [p.detach().cpu().clone() for p in pools], 0

    def pages(self, n):
        return -(-n // self.page)

    def free_pages(self):
        return [p for p, r in enumerate(self.ref) if r <= 0]

    def grow(self, n_new):
        free, short, cap = self.free_pages(), False, len(self.table[0]) * self.page
        for b, n in enumerate(n_new):
            if self.len[b] < 0 or n < 0:
                self.status |= 1
                continue
            if self.len[b] + n > cap:
                self.status |= 4
                continue
            have = self.pages(self.len[b])
            need = self.pages(self.len[b] + n) - have
            if need > 0 and (short or need > len(free)):
                short, self.status = True, self.status | 4
                continue
            for i in range(need):
                p = free.pop(0)
                self.table[b][have + i], self.ref[p] = p, 1
            self.len[b] += n

    def fork(self, src, dst):
        B, before, free = len(self.len), list(self.len), self.free_pages()
        P, cap = len(self.ref), len(self.table[0]) * self.page
        for i, (s, d) in enumerate(zip(src, dst)):
            if not (0 <= s < B and 0 <= d < B) or not 0 <= before[s] <= cap:
                self.status |= 1
                continue
            if before[d] != 0 or d in dst[:i]:
                self.status |= 2
                continue
            whole, rest = divmod(before[s], self.page)
            if rest:
                if not free:
                    self.status |= 4
                    continue
                p = free.pop(0)
                self.ref[p] = 1
                last = self.table[s][whole]
                if 0 <= last < P:
                    for pool in self.pools:
                        pool[:, p] = pool[:, last]
                else:
                    self.status |= 1
                self.table[d][whole] = p
            for c in range(whole):
                p = self.table[d][c] = self.table[s][c]
                if 0 <= p < P:
                    self.ref[p] += 1
                else:
                    self.status |= 1
            self.len[d] = before[s]

    def free(self, seqs):
        for s in seqs:
            if not 0 <= s < len(self.len):
                self.status |= 1
                continue
            if self.len[s] > 0:
                for c in range(min(self.pages(self.len[s]), len(self.table[s]))):
                    p = self.table[s][c]
                    if 0 <= p < len(self.ref) and self.ref[p] > 0:
                        self.ref[p] -= 1
                    else:
                        self.status |= 1
                self.table[s] = [-1] * len(self.table[s])
            self.len[s] = 0

    def compact(self):
        live = sum(r > 0 for r in self.ref)
        to = [p for p in range(live) if self.ref[p] <= 0]
        frm = [p for p in range(live, len(self.ref)) if self.ref[p] > 0]
        where = dict(zip(frm, to))
        for f, t in where.items():
            self.ref[t], self.ref[f] = self.ref[f], 0
            for pool in self.pools:
                pool[:, t] = pool[:, f]
        for b, n in enumerate(self.len):
            for c in range(min(self.pages(max(n, 0)), len(self.table[b]))):
                self.table[b][c] = where.get(self.table[b][c], self.table[b][c])
        return live
