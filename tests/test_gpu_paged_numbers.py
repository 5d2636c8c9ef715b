"""The numbers of the paged attention on the GPU: the weights' bits, their tail, scores far from 0 and
values that are not finite, each for every number of rows that a workgroup holds."""
from __future__ import annotations

import math

import pytest
import torch

import ytensor_amd as yt
from paged_ref import HALF_STEP, path_of
from test_gpu_paged import DT, cache, compare, ints, tokens, tree

pytestmark = pytest.mark.gpu
# (query heads a KV head, new tokens): 16, 32, 64 and 128 rows a workgroup
SHAPES = [(4, 1), (2, 16), (3, 21), (2, 60)]
# a weight is kept as two numbers of V's type: off by at most this of itself (bf16: a remainder below 2^-7
# of it, kept to 8 bits, is off by 2^-16; f16: below 2^-9, kept to 11 bits, 2^-21; f32 as it is)
WEIGHT = {torch.float32: 0.0, torch.float16: 2.0 ** -21, torch.bfloat16: 2.0 ** -16}


def bound(o, av, S, d, n, v_max, dt):
    """The result rounded once, the weights off by WEIGHT each in the product and in their sum, fp32 for the rest:
    a score of d products off by (d + 3) 2^-24 S, an exponential by 2^-22, the sums over n keys by n 2^-24, each in
    numerator and denominator; and a weight in float16, held 2^14 times as large, by 2^-25 of that unit."""
    tol = HALF_STEP[dt] * o.abs() + WEIGHT[dt] * (av + o.abs()) + 2.0 ** -24 * (2 * (d + 3) * S + 8 + 2 * n) * av
    if dt == torch.float16:
        tol = tol + 2.0 ** -25 + 2.0 ** -38 * n * v_max  # (the first: a result among float16's subnormals)
    return 1.01 * tol


def formula(q, rows_k, rows_v, kn, vn, parents, scale=None):
    """(out, bound) in 64 bits of one sequence, KV head by KV head: q [Hq, T, d], rows [Hkv, n, d], kn [Hkv, T, d]."""
    Hq, T, d = q.shape
    Hkv, dt = rows_k.shape[0], q.dtype
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    q, rows_k, rows_v, kn, vn = (x.cpu().double() for x in (q, rows_k, rows_v, kn, vn))
    out, tol = torch.zeros(Hq, T, d, dtype=torch.float64), torch.zeros(Hq, T, d, dtype=torch.float64)
    for h in range(Hkv):
        for t in range(T):
            at = path_of(parents, t)
            k, v = torch.cat([rows_k[h], kn[h, at]]), torch.cat([rows_v[h], vn[h, at]])
            for hq in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                s = scale * (k @ q[hq, t])
                p = torch.softmax(s, 0)
                o, av = p @ v, p @ v.abs()
                S = (abs(scale) * (k.abs() @ q[hq, t].abs())).max()
                out[hq, t], tol[hq, t] = o, bound(o, av, S, d, len(k), v.abs().max(), dt)
    return out, tol


def rows_of(pool, table, n):
    """A sequence's rows [Hkv, n, d] side by side."""
    page = pool.shape[2]
    return pool[table[: -(-n // page)].long()].transpose(0, 1).flatten(1, 2)[:, :n]


@pytest.mark.parametrize("n", [40, 1500])
@pytest.mark.parametrize("G,T", SHAPES)
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f16", 128), ("bf16", 64), ("f32", 64)])
def test_weights_keep_their_bits(dtype, d, G, T, n):
    """16-bit inputs: the weights are not rounded to 16 bits, so the result is off by its own rounding."""
    dt, Hkv, page = DT[dtype], 2, 16
    g, kp, vp, table, kv_len = cache(n + T, [n], Hkv, page, d, dt)
    q, kn, vn = tokens(g, 1, Hkv * G, Hkv, T, d, dt)
    parents = tree(g, 1, T)
    want, tol = formula(q[0], rows_of(kp, table[0], n), rows_of(vp, table[0], n), kn[0], vn[0], parents[0].tolist())
    compare(yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, parents=parents)[0], want, tol)
    sums = torch.nan_to_num(kp.float()).sum(2)
    out, _ = yt.paged_sparse_attention(q, kn, vn, kp, vp, sums, table, kv_len, -(-n // page), parents=parents)
    compare(out[0], want, tol)


@pytest.mark.parametrize("n", [200, 6000])
@pytest.mark.parametrize("G,T", SHAPES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_the_tail_behind_a_large_weight(dtype, G, T, n):
    """A key whose score is 17.5 nats above all others', and has no value: what the others bring is not lost,
    wherever the sequence is cut."""
    dt, Hkv, page, d = DT[dtype], 1, 16, 64
    g, kp, vp, table, kv_len = cache(n, [n], Hkv, page, d, dt)
    q, kn, vn = tokens(g, 1, G, Hkv, T, d, dt)
    q[:], kn[:], vn[:] = 0.0, 0.0, 0.0
    q[..., 0] = 10.0
    kp[:], vp[:] = 0.0, (4096 * (1 + torch.rand(vp.shape, generator=g))).to(dt).cuda()
    for row in (0, n // 2, n - 1):
        k, v = kp.clone(), vp.clone()
        k[table[0, row // page].long(), :, row % page, 0] = 14.0  # 10 * 14 / 8
        v[table[0, row // page].long(), :, row % page] = 0.0
        out = yt.paged_attention(q, kn, vn, k, v, table, kv_len)[0]
        want, tol = formula(q[0], rows_of(k, table[0], n), rows_of(v, table[0], n), kn[0], vn[0], None)
        compare(out, want, tol)


@pytest.mark.parametrize("n", [30, 2500])
@pytest.mark.parametrize("G,T", SHAPES)
@pytest.mark.parametrize("dtype,size", [("bf16", 3e4), ("f16", 2e4), ("f32", 1e12)])
def test_scores_far_from_zero(dtype, size, G, T, n):
    """Scores whose last bit is worth more than an exponential can hold: equal ones weigh the same, the largest
    takes all."""
    dt, Hkv, page, d = DT[dtype], 1, 16, 64
    g, kp, vp, table, kv_len = cache(n, [n], Hkv, page, d, dt)
    q, kn, vn = tokens(g, 1, G, Hkv, T, d, dt)
    side = size * (1 + torch.arange(d) / 100.0)  # no power of two, so that the scaled score is rounded
    q[:], kn[:], kp[:] = side.to(dt).cuda(), side.to(dt).cuda(), side.to(dt).cuda()
    for sign in (1.0, -1.0):
        out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len, scale=sign / 8)[0].cpu().double()
        v = rows_of(vp, table[0], n)[0].cpu().double()
        for t in range(T):
            all_v = torch.cat([v, vn[0, 0, : t + 1].cpu().double()])
            mean = all_v.mean(0)
            tol = bound(mean, all_v.abs().mean(0), 0.0, d, len(all_v), all_v.abs().max(), dt)
            assert ((out[:, t] - mean).abs() <= tol).all(), (sign, t)
    row = n // 3
    kp[table[0, row // page].long(), :, row % page] *= 1.25
    out = yt.paged_attention(q, kn, vn, kp, vp, table, kv_len)[0]
    one = rows_of(vp, table[0], n)[0, row]
    assert (out == one).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("G,T", [(4, 3), (2, 16), (3, 21), (2, 60)])
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f16", 128), ("bf16", 64), ("f32", 64), ("f32", 128)])
def test_values_that_are_not_finite(dtype, d, G, T, bad):
    """In V of a cached row they reach every query, in that of a new token those whose path holds it, each in its own
    element alone."""
    dt, Hkv, page, n = DT[dtype], 1, 16, 50
    g, kp, vp, table, kv_len = cache(T, [n], Hkv, page, d, dt)
    q, kn, vn = tokens(g, 1, G, Hkv, T, d, dt)
    parents = tree(g, 1, T)
    up = parents[0].tolist()
    hurt = T // 2
    sees = torch.tensor([hurt in path_of(up, t) for t in range(T)])
    assert sees.any() and not sees.all()
    v2, vn2 = vp.clone(), vn.clone()
    vn2[0, 0, hurt, 5::7] = bad
    v2[table[0, 1].long(), 0, 3, 2::9] = bad
    v2[table[0, 1].long(), 0, 4, 2::18] = bad  # the same sign twice
    want, tol = formula(q[0], rows_of(kp, table[0], n), rows_of(vp, table[0], n), kn[0], vn[0], up)
    out = yt.paged_attention(q, kn, vn2, kp, v2, table, kv_len, parents=parents)[0].cpu().double()
    reached = torch.zeros(T, d, dtype=torch.bool)
    reached[:, 2::9] = True
    reached[sees, 5::7] = True
    reached = reached.expand(G, T, d)
    odd = out[reached]
    assert (torch.isnan(odd) if math.isnan(bad) else odd == bad).all()
    compare(torch.where(reached, want, out), want, tol)


def test_a_value_that_is_not_finite_under_the_whole_weight():
    """One key, whose weight is 1."""
    for dt in DT.values():
        g, kp, vp, table, kv_len = cache(1, [1], 1, 16, 64, dt)
        q, _, _ = tokens(g, 1, 2, 1, 1, 64, dt)
        vp[table[0, 0].long(), 0, 0, ::2] = -math.inf
        out = yt.paged_attention(q, None, None, kp, vp, table, kv_len)
        assert (out[..., ::2] == -math.inf).all()
        assert torch.equal(out[0, 1, 0, 1::2], vp[table[0, 0].long(), 0, 0, 1::2])
