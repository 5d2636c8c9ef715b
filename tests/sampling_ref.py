"""The end of a drafted step in 64 bits and plain Python: what include/ythip.h says of ythip_verify_drafts, token by token."""
from __future__ import annotations

import math

import torch


def mass(x: float) -> float:
    return x if 0.0 < x < math.inf else 0.0


def masses(row):
    return torch.where((row > 0) & (row < math.inf), row, 0.0)


def draw(weights, x):
    """The first entry at which the sum passes x times all; -1 without a weight."""
    w = masses(weights)
    cum = torch.cumsum(w, 0)
    if not cum[-1] > 0:
        return -1
    hit = torch.nonzero(cum > x * cum[-1])
    return int(hit[0]) if len(hit) else int(torch.nonzero(w > 0)[-1])


def verify(target, tokens, u, u_next, draft=None, parents=None, tree_len=None):
    """(path, kept, next) as lists."""
    B, T, V = target.shape
    target, tokens, u, u_next = target.cpu().double(), tokens.cpu().tolist(), u.cpu().tolist(), u_next.cpu().tolist()
    draft = None if draft is None else draft.cpu().double()
    parents = [[t - 1 for t in range(T)]] * B if parents is None else parents.cpu().tolist()
    tree_len = [T] * B if tree_len is None else tree_len.cpu().tolist()
    paths, counts, nexts = [], [], []
    for b in range(B):
        tn = min(max(tree_len[b], 0), T)
        path = [0] if tn else []
        rest = None
        while path:
            n = path[-1]
            row = target[b, n]
            if draft is not None:
                t = n + 1
                if t >= tn:
                    break
                x = tokens[b][t]
                q = float(draft[b, t, x]) if 0 <= x < V else 0.0
                if 0 <= x < V and u[b][t] * q < mass(float(row[x])):
                    path.append(t)
                    continue
                left = (masses(row) - masses(draft[b, t])).clamp(min=0.0)
            else:
                kids = [t for t in range(n + 1, tn) if parents[b][t] == n and 0 <= tokens[b][t] < V]
                low, met, went = 0.0, set(), None
                for t in kids:
                    x = tokens[b][t]
                    high = low + (mass(float(row[x])) if x not in met else 0.0)
                    met.add(x)
                    if low <= u[b][n] < high:
                        went = t
                        break
                    low = high
                if went is not None:
                    path.append(went)
                    continue
                left = row.clone()
                left[list(met)] = 0.0
                left = masses(left)
            rest = left if (left > 0).any() else None
            break
        paths.append(path + [-1] * (T - len(path)))
        counts.append(len(path))
        nexts.append(-1 if not path else draw(rest if rest is not None else target[b, path[-1]], u_next[b]))
    return paths, counts, nexts
