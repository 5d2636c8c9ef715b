"""Windows where query rows alone fill the card: each workgroup then has a whole sequence's window for its rows, cached pages
of q's type and of 4 bits alike. A few sequences and heads of each batch, against window_ref (64 bits)."""
from __future__ import annotations

import math

import pytest
import torch

import q4_ref
import ytensor_amd as yt
from test_gpu_q4 import cache4, rows4
from test_gpu_window import DT, cache, ints, tokens, tree
from window_ref import Rows, attention

pytestmark = pytest.mark.gpu


class Some:
    """The rows of a few heads."""

    def __init__(self, rows, heads):
        self.rows, self.pick, self.heads = rows, heads, len(heads)

    def __call__(self, b, h):
        return self.rows(b, self.pick[h])


def check(out, before, q, kn, vn, rows_of, kv_len, parents, tree_len, window, sinks, seqs, heads, G):
    """rows_of(seqs): the cached rows of these sequences. Within the bound, NaN exactly where a token sees one, and as it was
    behind the last token."""
    hq = [h * G + g for h in heads for g in range(G)]
    part = lambda t, hs: None if t is None else t[seqs][:, hs]  # noqa: E731
    sub = lambda t: None if t is None else t[seqs]  # noqa: E731
    want, tol = attention(part(q, hq), part(kn, heads), part(vn, heads), Some(rows_of(seqs), heads), kv_len[seqs], sub(parents),
                          sub(tree_len), window, sinks)
    got, was = part(out, hq).cpu(), part(before, hq).cpu()
    worst, nans = 0.0, 0
    for i in range(len(seqs)):
        n = int(tree_len[seqs[i]])
        o, w, t = got[i, :, :n].double(), want[i, :, :n], tol[i, :, :n]
        assert torch.equal(o.isnan(), w.isnan())
        real = ~w.isnan()
        nans += int((~real).sum())
        assert torch.isfinite(o[real]).all()
        if real.any():
            # (a row that sees a NaN has no bound where its other channels have values: that of its own size)
            worst = max(worst, ((o - w).abs()[real] / t[real].nan_to_num(math.inf).clamp(min=1e-300)).max().item())
        assert torch.equal(got[i, :, n:], was[i, :, n:])
    print(f"worst error / bound {worst:.3f}, {nans} NaN", flush=True)
    assert worst <= 1.0
    return nans


SHAPES = [  # B, Hkv, G, T, page
    (8, 8, 2, 130, 32),    # 64 query rows a workgroup
    (16, 8, 4, 128, 16),   # 128
    (32, 8, 1, 200, 64),   # 128, of two tiles the second in part
]


@pytest.mark.parametrize("B,Hkv,G,T,page", SHAPES)
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 64), ("f16", 128), ("f32", 64), ("f32", 128)])
@pytest.mark.parametrize("kind,window,sinks", [("chain", 200, 0), ("tree", 333, 5), ("chain", 90, 700), ("tree", 60, 100)])
def test_pages_of_values(dtype, d, B, Hkv, G, T, page, kind, window, sinks):
    dt = DT[dtype]
    lens = [1000 - 333 * (b % 4) for b in range(B)]
    assert yt.paged_workspace_bytes(dt, B, Hkv * G, Hkv, T, d, -(-1000 // page) + 1, page, window=window, sinks=sinks) == 0
    g, kp, vp, table, kv_len = cache(T, lens, Hkv, page, d, dt)
    assert table.shape[1] == -(-1000 // page) + 1
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    parents = tree(g, B, T) if kind == "tree" else None
    tree_len = ints([T - 7 * (b % 3) for b in range(B)])
    # a V and a K that are no number, near the end of the cache: the first tokens see them, the last ones do not
    for b in range(B):
        r = lens[b] + 40 - window
        if r >= 0:
            p = int(table[b, r // page])
            vp[p, 0, r % page, 3] = math.nan
            kp[p, 1, r % page, 5] = math.nan
    out = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
    before = out.clone()
    yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents, tree_len=tree_len, out=out, window=window, sinks=sinks)
    rows = lambda seqs: Rows(kp, vp, table[seqs], kv_len[seqs])  # noqa: E731
    assert check(out, before, q, kn, vn, rows, kv_len, parents, tree_len, window, sinks, [0, 3, B - 1], [0, 1, Hkv - 1], G) > 0


@pytest.mark.parametrize("B,Hkv,G,T,page", SHAPES)
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 64), ("f16", 128), ("f32", 64)])
@pytest.mark.parametrize("kind,window,sinks", [("chain", 200, 0), ("tree", 333, 5), ("chain", 90, 700), ("tree", 60, 100)])
def test_pages_in_4_bits(dtype, d, B, Hkv, G, T, page, kind, window, sinks):
    dt = DT[dtype]
    lens = [1000 - 333 * (b % 4) for b in range(B)]
    assert yt.paged_q4_workspace_bytes(dt, B, Hkv * G, Hkv, T, d, -(-1000 // page) + 1, page, window=window, sinks=sinks) == 0
    g, kp, vp, table, kv_len = cache4(T, lens, Hkv, page, d, dt)
    q, kn, vn = tokens(g, B, Hkv * G, Hkv, T, d, dt)
    parents = tree(g, B, T) if kind == "tree" else None
    tree_len = ints([T - 7 * (b % 3) for b in range(B)])
    for b in range(B):
        r = lens[b] + 40 - window
        if r >= 0:
            p = int(table[b, r // page])
            vp[p, 0, q4_ref.place(page, d, r % page, 3, "v")[2]] = 255
            kp[p, 1, q4_ref.place(page, d, r % page, 5, "k")[2]] = 255
    out = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
    before = out.clone()
    yt.paged_attention_q4(q, kn, vn, kp, vp, table, kv_len, page, parents=parents, tree_len=tree_len, out=out, window=window, sinks=sinks)
    rows = lambda seqs: rows4(kp, vp, table[seqs], kv_len[seqs], page, d)  # noqa: E731
    assert check(out, before, q, kn, vn, rows, kv_len, parents, tree_len, window, sinks, [0, 3, B - 1], [0, 1, Hkv - 1], G) > 0
