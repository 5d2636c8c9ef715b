"""Probabilities and the verification of drafted tokens on the GPU, against 64 bits (sampling_ref)."""
from __future__ import annotations

import math

import pytest
import torch

import ytensor_amd as yt
from sampling_ref import verify as model

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_probs(p, logits, temperature):
    """p = w / sum: a difference of two logits is half a step off (|d| / T 2^-24 of w), an exponential and the roundings
    around it 4 steps of 2^-23; the sum of n positive numbers is off by a step of 2^-24 for each that a thread of 256 adds
    and 40 for the joining (each of them two exponentials' products, 2^-21); numbers below 2^-126 may vanish."""
    x = logits.detach().cpu().double()
    n = x.shape[-1]
    want = torch.softmax(x / temperature, -1)
    d = (x.amax(-1, keepdim=True) - x).clamp(max=200 * temperature) / temperature
    tol = want * (2.0 ** -24 * d + 2.0 ** -21 + 2.0 ** -24 * (n / 256 + 8) + 40 * 2.0 ** -21) + 2.0 ** -125
    off = (p.cpu().double() - want).abs()
    print(f"worst error / bound {(off / tol).max().item():.3f}", flush=True)
    assert (off <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,n,temperature", [(1, 1, 1.0), (2, 7, 0.5), (1, 4097, 1.3), (3, 9001, 0.7), (1, 151936, 1.0),
                                                (200, 33, 1.0), (193, 5003, 0.3), (17, 50257, 1.0), (191, 8192, 2.0)])
def test_probs(dtype, rows, n, temperature):
    x = (4.0 * torch.randn(rows, n, generator=torch.Generator().manual_seed(rows + n))).to(DT[dtype]).cuda()
    check_probs(yt.token_probs(x, temperature), x, temperature)


@pytest.mark.parametrize("n", [100, 20000])
def test_probs_of_strided_rows(n):
    """Rows at an odd stride and address, of a transposed tensor, and into a given output, whose other elements stay."""
    base = torch.randn(5, n + 3, generator=torch.Generator().manual_seed(n)).to(torch.bfloat16).cuda()
    out = torch.full((5, n + 5), 7.0, device="cuda")
    got = yt.token_probs(base[:, 3:], 1.0, out=out[:, 1:n + 1])
    assert got.data_ptr() == out.data_ptr() + 4
    check_probs(got, base[:, 3:], 1.0)
    assert (out[:, 0] == 7).all() and (out[:, n + 1:] == 7).all()
    turned = base.t().contiguous().t()
    check_probs(yt.token_probs(turned, 1.0), turned, 1.0)
    check_probs(yt.token_probs(base[0], 1.0), base[0], 1.0)
    three = base[:4, :n].unflatten(0, (2, 2))
    check_probs(yt.token_probs(three, 1.0), three, 1.0)
    assert yt.token_probs(base[:0]).shape == (0, n + 3) and yt.token_probs(base[:, :0]).shape == (5, 0)
    with pytest.raises(ValueError):
        yt.token_probs(base, out=torch.empty(n + 3, 5, device="cuda").t())
    with pytest.raises(ValueError):
        yt.token_probs(base, out=torch.empty_like(base))


@pytest.mark.parametrize("n", [65, 30000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_probs_of_rows_with_infinities(dtype, n):
    x = torch.randn(6, n, generator=torch.Generator().manual_seed(1)).to(DT[dtype])
    x[0, 1:] = -math.inf
    x[1] = -math.inf
    x[2, n - 2] = math.inf
    x[3, n // 2] = math.nan
    x[4, ::2] = -math.inf
    x[5] = torch.finfo(DT[dtype]).min
    x[5, 3] = torch.finfo(DT[dtype]).max
    p = yt.token_probs(x.cuda(), 1.0).cpu()
    assert p[0, 0] == 1 and (p[0, 1:] == 0).all() and (p[1] == 0).all() and p[2:4].isnan().all()
    assert (p[4, ::2] == 0).all() and abs(p[4].double().sum() - 1) < 1e-4
    assert p[5, 3] == 1 and p[5].sum() == 1


@pytest.mark.parametrize("dtype,n", [("bf16", 8191), ("bf16", 155648), ("f16", 155661), ("bf16", 170003), ("f32", 73731), ("f32", 73728), ("f32", 100007)])
def test_probs_of_many_rows(dtype, n):
    """Rows with a workgroup each: within what its registers hold, to the last of it, and beyond; at an odd stride too."""
    x = (3.0 * torch.randn(8, n, generator=torch.Generator().manual_seed(n))).to(DT[dtype])
    x[1, n - 1] = math.inf
    x[2, n - 1] = math.nan
    x[3] = -math.inf
    x[4, : n - 3] = -math.inf
    x[5, n - 9] = 60.0
    for wide in (0, 1):
        rows = torch.zeros(200, n + wide, dtype=DT[dtype])
        rows[:, :n] = x.repeat(25, 1)
        p = yt.token_probs(rows.cuda()[:, :n], 0.7).cpu()
        assert p[1:3].isnan().all() and (p[3] == 0).all() and (p[4, : n - 3] == 0).all()
        for r in (0, 4, 5, 6, 7):
            check_probs(p[r], x[r], 0.7)
        assert torch.equal(p.view(25, 8, n).view(torch.int32), p[:8].view(torch.int32).expand(25, 8, n))


def drafts(seed, B, T, V, dtype, chain, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = spread * torch.randn(B, T, V, generator=g)
    target = torch.softmax(logits, -1)
    near = torch.softmax(logits + 0.7 * torch.randn(B, T, V, generator=g), -1)
    above = torch.arange(-1, T - 1).clamp(min=0).expand(B, T)
    if not chain:
        above = torch.clamp(torch.arange(T)[None] - torch.randint(1, 4, (B, T), generator=g), min=0)
    near = torch.gather(near, 1, above[..., None].expand(B, T, V)).contiguous()
    tokens = torch.multinomial(near.reshape(-1, V), 1, generator=g).reshape(B, T).int()
    u, un = torch.rand(B, T, generator=g), torch.rand(B, generator=g)
    dt = DT[dtype]
    return (target.to(dt).cuda(), tokens.cuda(), u.cuda(), un.cuda()), near.to(dt).cuda(), above.int().cuda()


def check(args, **kw):
    got = yt.verify_drafts(*args, **kw)
    want = model(*args, **{k: v for k, v in kw.items() if k in ("draft", "parents", "tree_len")})
    print("kept", want[1], flush=True)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].tolist() == want[2]
    return want


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 2, 7), (2, 6, 4096), (5, 17, 4097), (1, 64, 9000), (2, 70, 333), (4, 5, 20001)])
@pytest.mark.parametrize("kind", ["draft", "chain", "tree"])
def test_verify(kind, B, T, V, dtype):
    for seed in range(3):
        args, near, above = drafts(100 * seed + T, B, T, V, dtype, kind != "tree", spread=(3.0, 6.0, 1.0)[seed])
        check(args, draft=near if kind == "draft" else None, parents=above if kind == "tree" else None,
              tree_len=ints([max(0, T - b) for b in range(B)]) if seed else None)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["draft", "chain", "tree"])
@pytest.mark.parametrize("V", [(1 << 18) - 5, 1 << 18, (1 << 18) + 1, 300007])
def test_verify_of_long_rows(kind, V, dtype):
    """Rows of more runs than lanes, whole and not."""
    args, near, above = drafts(V, 2, 4, V, dtype, kind != "tree", spread=2.0)
    for u_next in (args[3], torch.tensor([0.0, 1 - 2.0 ** -24], device="cuda")):
        check((*args[:3], u_next), draft=near if kind == "draft" else None, parents=above if kind == "tree" else None)


@pytest.mark.parametrize("kind", ["draft", "chain", "tree"])
def test_verify_keeps_long_paths(kind):
    """A target that is all but sure of the drafted tokens, up to the last of 1024."""
    T, V = 1024, 40
    args, near, above = drafts(5, 2, T, V, "f32", kind != "tree")
    target, tokens = args[0], args[1].long()
    sure = torch.full_like(target, 0.001 / V)
    up = above.long() if kind == "tree" else torch.arange(-1, T - 1, device="cuda").clamp(min=0).expand(2, T)
    for t in range(T - 1, 0, -1):  # the first child of a token last, so that it stays
        for b in range(2):
            sure[b, up[b, t]] = 0.001 / V
            sure[b, up[b, t], tokens[b, t]] = 0.999
    args = (sure.contiguous(), *args[1:])
    want = check(args, draft=near if kind == "draft" else None, parents=above if kind == "tree" else None)
    assert max(want[1]) > (3 if kind == "tree" else 64)  # (a first child's line soon has no children in such a tree)


@pytest.mark.parametrize("T", [65, 130, 1023])
def test_verify_of_a_comb(T):
    """Every second token goes on, behind a sibling that is not kept: a path over many runs of 64 tokens."""
    V, t = 50, torch.arange(T)
    parents = torch.where(t % 2 == 1, t - 1, t - 2).clamp(min=-1).int().expand(2, T).contiguous().cuda()
    tokens = torch.where(t % 2 == 1, 3, 5).int().expand(2, T).contiguous().cuda()
    p = torch.full((2, T, V), 0.01 / V)
    p[..., 3], p[..., 5] = 0.2, 0.79
    u = torch.full((2, T), 0.6)
    u[1, T // 4 * 2] = 0.1
    want = check((p.cuda(), tokens, u.cuda(), torch.tensor([0.5, 0.999]).cuda()), parents=parents)
    assert want[1][0] == (T + 1) // 2


def test_verify_of_siblings_with_one_token_and_bad_tokens():
    """Of two siblings with one token the first has its probability; tokens and parents out of range are never kept, and
    what hangs below them is not reached."""
    p = torch.tensor([0.1, 0.2, 0.3, 0.4]).expand(1, 7, 4).contiguous().cuda()
    tokens = ints([[0, 3, 3, -1, 4, 1, 2]])
    parents = ints([[-1, 0, 0, 0, 0, 0, 3]])
    for a in (0.0, 0.39, 0.41, 0.59, 0.61, 0.99):
        for c in (0.0, 0.3, 0.4, 0.999):
            u = torch.full((1, 7), a, device="cuda")
            check((p, tokens, u, torch.tensor([c], device="cuda")), parents=parents)
            check((p, tokens, u, torch.tensor([c], device="cuda")), parents=ints([[5, 7, 1, -1, 9, 0, 2]]))


@pytest.mark.parametrize("V", [5000, 270000])
@pytest.mark.parametrize("kind", ["draft", "tree"])
def test_verify_where_nothing_is_left(kind, V):
    """A draft row that is the target's, a node whose children hold all of it, rows without a weight, with NaN, negative
    and infinite entries, and random numbers of 0, all but 1, 1 and NaN."""
    target = torch.zeros(6, 3, V)
    target[:, :, 7], target[:, :, 4500] = 0.25, 0.75
    target[3] = 0.0
    target[4, :, 10:40] = torch.tensor([math.nan, -1.0, math.inf]).repeat(10)
    target[5, 2] = math.nan
    tokens = ints([[0, 7, 4500]]).expand(6, 3).contiguous()
    near = target.clone()
    near[0, :, 7] = 1.0
    near[2, :, 4500] = math.inf
    for x in (0.0, 0.2499999, 0.5, 1 - 2.0 ** -24, 1.0, math.nan):
        u = torch.tensor([[x, 0.999, 0.999]], device="cuda").expand(6, 3).contiguous()
        un = torch.full((6,), x, device="cuda")
        kw = dict(draft=near.cuda()) if kind == "draft" else dict(parents=ints([[-1, 0, 0]]).expand(6, 3).contiguous())
        check((target.cuda(), tokens, u, un), **kw)


def test_verify_of_strided_rows():
    """Every second row of wider tensors at an odd address, and a target whose vocabulary is not contiguous."""
    (target, tokens, u, un), near, _ = drafts(9, 2, 5, 1001, "bf16", True)
    wide = torch.full((2, 10, 1007), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, ::2, 5:1006] = target
    check((wide[:, ::2, 5:1006], tokens, u, un), draft=near)
    check((target.transpose(1, 2).contiguous().transpose(1, 2), tokens, u, un))
    spread = torch.zeros(2, 10, dtype=torch.int32, device="cuda")
    spread[:, ::2] = tokens
    out = (ints([[5] * 5] * 2), ints([5, 5]), ints([5, 5]))
    got = yt.verify_drafts(target, spread[:, ::2], u, un, draft=near, out=out)
    assert all(a is b for a, b in zip(got, out))
    want = model(target, tokens, u, un, draft=near)
    assert [x.tolist() for x in got] == [want[0], want[1], want[2]]
    with pytest.raises(ValueError):
        yt.verify_drafts(target, tokens, u, un, draft=near, parents=tokens)
    with pytest.raises(ValueError):
        yt.verify_drafts(target, tokens, u.double(), un)
    with pytest.raises(ValueError):
        yt.verify_drafts(target, tokens, u, un, draft=near.float())
    with pytest.raises(ValueError):
        yt.verify_drafts(target, tokens, u, un, out=(out[0].t().contiguous().t(), *out[1:]))


def test_a_captured_step():
    """Probabilities and verification in one HIP graph, replayed with other logits, tokens and random numbers."""
    B, T, V = 3, 6, 12345
    logits = torch.zeros(B, T, V, dtype=torch.bfloat16, device="cuda")
    _, _, above = drafts(1, B, T, V, "f32", False)
    tokens, u, un = ints([[0] * T] * B), torch.zeros(B, T, device="cuda"), torch.zeros(B, device="cuda")
    lens = ints([6, 5, 0])
    p = yt.token_probs(logits, 0.8)
    out = yt.verify_drafts(p, tokens, u, un, parents=above, tree_len=lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yt.token_probs(logits, 0.8, out=p)
        yt.verify_drafts(p, tokens, u, un, parents=above, tree_len=lens, out=out)
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        logits.copy_(4.0 * torch.randn(B, T, V, generator=g))
        best = torch.gather(logits.float(), 1, above.long()[..., None].expand(B, T, V)).argmax(-1).int()
        tokens.copy_(best)
        u.copy_(torch.rand(B, T, generator=g) * 0.3)
        un.copy_(torch.rand(B, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        check_probs(p, logits, 0.8)
        want = model(p, tokens, u, un, parents=above, tree_len=lens)
        assert [x.tolist() for x in out] == [want[0], want[1], want[2]]


def test_two_streams_at_once():
    """Steps on two streams that overlap: what each gives alone, bit for bit."""
    B, T, V = 4, 5, 60001
    steps = []
    for seed in range(2):
        (_, tokens, u, un), _, above = drafts(seed, B, T, V, "f32", False)
        logits = torch.randn(B, T, V, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()

        def step(logits=logits, tokens=tokens, u=u, un=un, above=above):
            p = yt.token_probs(logits, 0.5)
            return (p, *yt.verify_drafts(p, tokens, u, un, parents=above))
        steps.append((step, step()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for st, (step, _) in zip(streams, steps):
            with torch.cuda.stream(st):
                got.append(step())
        torch.cuda.synchronize()
        for out, (_, want) in zip(got, steps):
            assert all(torch.equal(x, y) for x, y in zip(out, want))
