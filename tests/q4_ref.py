"""4-bit pages in 64 bits and plain loops over groups: what include/ythip.h says of them."""
from __future__ import annotations

import math

import torch

STEPS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def group(x, dtype):
    """(32 codes, scale byte) of 32 numbers."""
    top = max(abs(v) for v in x)
    if any(math.isnan(v) for v in x) or math.isinf(top):
        return [0] * 32, 255  # (the codes of a group without a value do not count)
    e = -125
    while e < (13 if dtype == torch.float16 else 125) and top > 7 * 2.0 ** e:
        e += 1
    codes = []
    for v in x:
        a = abs(v) / 2.0 ** e
        best = min(range(8), key=lambda i: (abs(a - STEPS[i]), i % 2))
        codes.append(best + (8 if math.copysign(1.0, v) < 0 else 0))
    return codes, e + 127


def rows(x):
    """(codes [n, d], scale bytes [n, d / 32]) of rows x [n, d]."""
    codes, scales = [], []
    for row in x.double().tolist():
        g = [group(row[i:i + 32], x.dtype) for i in range(0, len(row), 32)]
        codes.append([c for cs, _ in g for c in cs])
        scales.append([s for _, s in g])
    return torch.tensor(codes, dtype=torch.uint8), torch.tensor(scales, dtype=torch.uint8)


def place(page, d, r, ch, which):
    """(byte, half) of channel ch of row r in a block, and its scale's byte."""
    if which == "k":
        return (r * d + ch) // 2, ch % 2, page * d // 2 + r * (d // 32) + ch // 32
    per = d // 16
    return ((r // 8 * 16 + ch // per) * 8 + r % 8) * (d // 32) + ch % per // 2, ch % 2, page * d // 2 + (r // 8 * (d // 32) + ch // 32) * 8 + r % 8


def _maps(page, d, which):
    at = torch.empty(page, d, dtype=torch.int64)
    half = torch.empty(page, d, dtype=torch.int64)
    scale = torch.empty(page, d, dtype=torch.int64)
    for r in range(page):
        for ch in range(d):
            at[r, ch], half[r, ch], scale[r, ch] = place(page, d, r, ch, which)
    return at, half, scale


_cache = {}


def maps(page, d, which):
    if (page, d, which) not in _cache:
        _cache[page, d, which] = _maps(page, d, which)
    return _cache[page, d, which]


def put(block, r, codes, scales, page, d, which):
    """One row's codes [d] and scale bytes [d / 32] into a block (bytes, in place)."""
    for ch in range(d):
        at, half, sc = place(page, d, r, ch, which)
        block[at] = (int(block[at]) & (15 << 4 * (1 - half))) | int(codes[ch]) << 4 * half
        block[sc] = int(scales[ch // 32])


def values(blocks, page, d, which):
    """float64 [..., page, d] that blocks [..., bytes] hold."""
    at, half, scale = maps(page, d, which)
    b = blocks.cpu().long()
    code = b[..., at] >> (4 * half) & 15
    v = torch.tensor(STEPS + [-s for s in STEPS], dtype=torch.float64)[code] * torch.exp2(b[..., scale].double() - 127)
    return torch.where(b[..., scale] == 255, math.nan, v)


def pack(x, which):
    """Rows x [..., page, d] as blocks [..., bytes], by whole tensors (checked against group() in the CPU tests)."""
    page, d = x.shape[-2:]
    g = x.double().unflatten(-1, (d // 32, 32))
    top = g.abs().amax(-1)
    e = torch.full_like(top, -125)
    for k in range(-125, 13 if x.dtype == torch.float16 else 125):
        e = torch.where(top > 7 * 2.0 ** k, k + 1.0, e)
    a = (g.abs() / torch.exp2(e)[..., None]).unsqueeze(-1)
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
    code = order[(a - torch.tensor(STEPS, dtype=torch.float64)[order]).abs().argmin(-1)]
    code = (code + 8 * torch.signbit(g).long()).flatten(-2)
    at, half, scale = maps(page, d, which)
    out = torch.zeros(*x.shape[:-2], page * (d // 2 + d // 32), dtype=torch.int64)
    lead = tuple(x.shape[:-2])
    out.scatter_add_(-1, at.flatten().expand(*lead, -1), (code << (4 * half)).flatten(-2))
    se = (e.long() + 127).repeat_interleave(32, -1)
    out.scatter_(-1, scale.flatten().expand(*lead, -1), se.flatten(-2))
    return out.to(torch.uint8)
