"""4-bit attention on the GPU where its numbers end: queries that are not finite, weights far below the largest, what two
pieces of a weight hold."""
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


def pool(k, v, page):
    """Rows k and v [B, Hkv, n, d] as 4-bit pools, a table and lengths, and the values that the pools hold."""
    B, Hkv, n, d = k.shape
    pages = max(1, -(-n // page))
    pools, values = [], []
    for x, which in ((k, "k"), (v, "v")):
        x = torch.nn.functional.pad(x, (0, 0, 0, pages * page - n))
        blocks = q4_ref.pack(x.unflatten(2, (pages, page)).transpose(1, 2).flatten(0, 1), which)
        pools.append(blocks.cuda())
        values.append(q4_ref.values(blocks, page, d, which))
    table, kv_len = ints([[b * pages + c for c in range(pages)] for b in range(B)]), ints([n] * B)
    return (*pools, table, kv_len), Rows(*values, table, kv_len)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f16", 128), ("f32", 64)])
@pytest.mark.parametrize("T", [1, 5, 40, 140])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_queries_with_an_infinity(dtype, d, T, sign):
    """One channel of a query is infinite, and every cached key is below 0 there: all scores are -inf, so the row is zero;
    with a new key above 0, or an infinity of the other sign, it is NaN. Other heads and tokens are as ever."""
    dt, page, n, Hq, c = DT[dtype], 16, 45, 3, 5
    g = torch.Generator().manual_seed(T + d)
    k, v = (torch.randn(1, 1, n, d, generator=g).to(dt) for _ in range(2))
    q, kn, vn = (torch.randn(1, h, T, d, generator=g).to(dt) for h in (Hq, 1, 1))
    k[..., c], kn[..., c] = -2.0, -1.0
    kn[0, 0, T // 2, c] = sign
    where = torch.zeros(1, Hq, T, dtype=torch.bool)
    where[0, 0, 0] = where[0, 1, T - 1] = where[0, 2, T // 2] = where[0, 2, 0] = True
    q[where] = torch.where(torch.arange(d) == c, torch.inf, q[where])
    q[0, 2, 0, c] = -torch.inf
    q, kn, vn = q.cuda(), kn.cuda(), vn.cuda()
    args, rows = pool(k, v, page)
    out = yt.paged_attention_q4(q, kn, vn, *args, page).cpu()
    want, tol = attention(q, kn, vn, rows, args[-1])
    assert want[0, 2, 0].isnan().all() and ((want[where] == 0) | want[where].isnan()).all()
    assert (want[0, 1, T - 1] == 0).all() == (sign < 0)
    assert torch.equal(want.isnan(), out.isnan())
    here = out[where].double()
    assert torch.equal(here[~here.isnan()], want[where][~want[where].isnan()])
    compare(out[~where], want[~where], tol[~where])


@pytest.mark.parametrize("window", [0, 1000])
@pytest.mark.parametrize("steps", [8.0, 16.0, 20.0, 24.0])
@pytest.mark.parametrize("T", [2, 66])
def test_float16_weights_over_pools_of_values(steps, T, window):
    """The same over float16 pools, whose weights have one unit: 21 bits of a weight, at best 2^-39 of the largest, so with
    |v| that much a key; the rest as there."""
    d, page, n = 64, 16, 40
    g = torch.Generator().manual_seed(T)
    q, kn, k = torch.zeros(1, 2, T, d), torch.zeros(1, 1, T, d), torch.zeros(1, 1, n, d)
    q[..., 0], kn[:, :, 0, 0] = 4.0, steps / 4.0
    vn, v = (40000.0 + 20000.0 * torch.rand(1, 1, m, d, generator=g) for m in (T, n))
    vn[:, :, 0] = 0.0
    q, kn, vn, k, v = (x.half() for x in (q, kn, vn, k, v))
    pad = lambda x: torch.nn.functional.pad(x[0, 0], (0, 0, 0, -n % page)).view(-1, 1, page, d).cuda()  # noqa: E731
    out = yt.paged_attention(q.cuda(), kn.cuda(), vn.cuda(), pad(k), pad(v), ints([list(range(-(-n // page)))]), ints([n]), scale=1.0,
                             window=window).cpu().double()
    values = torch.cat([vn[0, 0].double(), v[0, 0].double()])
    for t in range(T):
        keys = torch.cat([torch.arange(t + 1), T + torch.arange(n)])
        w = torch.where(keys == 0, 1.0, math.exp(-steps)).double()
        want = (w[:, None] * values[keys]).sum(0) / w.sum()
        off = 2.0 ** -21 + 2.0 ** -23 * (steps + 4) + 2.0 ** -24 * len(keys)
        tol = (2.0 ** -11 + off) * want + 2.0 ** -25 + 2.0 ** -39 * values[keys].sum(0)
        worst = ((out[0, :, t] - want).abs() / tol).max().item()
        assert worst <= 1.0, (t, worst)


@pytest.mark.parametrize("dtype,steps", [("f16", 20.0), ("f16", 27.75), ("f16", 31.0), ("bf16", 27.75), ("f32", 27.75)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T,n", [(9, 0), (66, 0), (200, 40)])
def test_weights_far_below_the_largest(dtype, steps, d, T, n):
    """The key with the largest weight has a V of 0: what the others add, e^-steps (2^-29, 2^-40, 2^-45) of it each, is all
    of the result. A weight keeps 16 bits (fp32: 24): 2^-16 (2^-24) of sum p |v|; a score of two products and its
    exponential are (steps + 4) 2^-23 off, a sum of n keys n 2^-24; the result is half a step of its type, at least of its
    smallest number. A new float16 token's weight is a float16 number times 2^25 and its largest is 1, so half a step of the
    smallest, 2^-24, is 2^-50: with |v| that much a key."""
    dt, page = DT[dtype], 16
    g = torch.Generator().manual_seed(T)
    q, kn, k = torch.zeros(1, 2, T, d), torch.zeros(1, 1, T, d), torch.zeros(1, 1, n, d)
    q[..., 0], kn[:, :, 0, 0] = 4.0, steps / 4.0
    vn, v = (40000.0 + 20000.0 * torch.rand(1, 1, m, d, generator=g) for m in (T, n))
    vn[:, :, 0] = 0.0
    q, kn, vn, k, v = (x.to(dt) for x in (q, kn, vn, k, v))
    args, rows = pool(k, v, page)
    out = yt.paged_attention_q4(q.cuda(), kn.cuda(), vn.cuda(), *args, page, scale=1.0).cpu().double()
    _, _, vc = rows(0, 0)
    values = torch.cat([vn[0, 0].double(), vc])
    f = torch.finfo(dt)
    least = f.smallest_normal * f.eps
    for t in range(T):
        keys = torch.cat([torch.arange(t + 1), T + torch.arange(n)])
        w = torch.where(keys == 0, 1.0, math.exp(-steps)).double()
        want = (w[:, None] * values[keys]).sum(0) / w.sum()
        off = 2.0 ** (-24 if dt == torch.float32 else -16) + 2.0 ** -23 * (steps + 4) + 2.0 ** -24 * len(keys)
        tol = (f.eps / 2 + off) * want + least / 2 + (2.0 ** -50 * values[keys].sum(0) if dt == torch.float16 else 0.0)
        worst = ((out[0, :, t] - want).abs() / tol).max().item()
        assert worst <= 1.0, (t, worst)


def cancelling(g, T, n, d, dt, scale):
    """One head: q, new rows and n cached ones, where each token's own V is such that its result is all but 0: what is
    left of it is the weights' error, for the result's own rounding is as small as the result."""
    q, k, v = torch.randn(T, d, generator=g).to(dt), torch.randn(n, d, generator=g).to(dt), torch.randn(n, d, generator=g).to(dt)
    # a score of log(n + t) + 1: a third or so of the weight is the token's own
    long = torch.log(n + 1.0 + torch.arange(T)).add(1)[:, None] / (scale * q.float().square().sum(-1, keepdim=True))
    kn, vn = (q.float() * long).to(dt), torch.zeros(T, d, dtype=dt)
    return q, k, v, kn, vn


@pytest.mark.parametrize("dtype,bits", [("bf16", 16), ("f16", 16), ("f32", 24)])
@pytest.mark.parametrize("T", [1, 10, 40, 140])
@pytest.mark.parametrize("d,pages", [(64, "4 bits"), (128, "4 bits"), (64, "values"), (128, "values")])
def test_weights_keep_their_bits(dtype, bits, T, d, pages):
    """Results that cancel, within 2^-bits of sum p |v| for the weights; a score and its exponential (d + 3) 2^-24 S and
    2^-22, S = scale sum |q k|, sums over n keys n 2^-24, each for the numerator and the denominator; half a step of the
    result. (With a weight's first 8 bits alone, or with the bits behind them of another key, it is 14 to 110 times the bound.)"""
    dt, page, n, scale = DT[dtype], 16, 37, 1.0 / math.sqrt(d)
    g = torch.Generator().manual_seed(10 * T + d)
    q, k, v, kn, vn = cancelling(g, T, n, d, dt, scale)
    if pages == "values":
        pad = lambda x: torch.nn.functional.pad(x, (0, 0, 0, -n % page)).view(-1, 1, page, d)  # noqa: E731
        pools = (pad(k).cuda(), pad(v).cuda(), ints([list(range(-(-n // page)))]), ints([n]))
        kc, vc = k.double(), v.double()
    else:
        pools, rows = pool(k[None, None], v[None, None], page)
        _, kc, vc = rows(0, 0)
    want, tol = torch.zeros(T, d, dtype=torch.float64), torch.zeros(T, d, dtype=torch.float64)
    for t in range(T):
        keys = torch.cat([kc, kn[:t + 1].double()])
        p = torch.softmax(scale * (keys @ q[t].double()), 0)
        vn[t] = (-(p[:-1] @ torch.cat([vc, vn[:t].double()])) / p[-1]).to(dt)
        values = torch.cat([vc, vn[:t + 1].double()])
        want[t] = p @ values
        S = (scale * (keys.abs() @ q[t].double().abs())).max()
        size = p @ values.abs()
        tol[t] = torch.finfo(dt).eps / 2 * want[t].abs() + size * (2.0 ** -bits + 2.0 ** -24 * (2 * (d + 3) * S + 8 + 2 * len(keys)))
    new = (q[None, None].cuda(), kn[None, None].cuda(), vn[None, None].cuda())
    if pages == "values":
        out = yt.paged_attention(*new, *pools)
    else:
        out = yt.paged_attention_q4(*new, *pools, page)
    worst = ((out[0, 0].cpu().double() - want).abs() / tol).max().item()
    print(f"worst error / bound {worst:.3f}, result / sum p |v| {(want.abs().max() / size.max()).item():.1e}", flush=True)
    assert worst <= 1.0
