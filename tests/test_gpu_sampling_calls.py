"""Calls of token_probs and verify_drafts on the GPU that their documentation allows and that are easily got wrong: layouts,
sizes, memory that arguments share."""
from __future__ import annotations

import pytest
import torch

import ytensor_amd as yt

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def logits(shape, dtype=torch.bfloat16, seed=0):
    return (3.0 * torch.randn(shape, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


@pytest.mark.parametrize("n", [1, 300, 20000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_probs_of_rows_that_share_memory(n, dtype):
    """One row expanded to several, a batch of one step for all sequences, overlapping rows: what a copy of them gives. An
    `out` of that kind cannot hold the result."""
    row = logits((1, n), dtype)
    x = logits((3, 1, n), dtype, 1)
    wide = logits((n + 5,), dtype, 2)
    for t in (row.expand(4, n), x.expand(3, 5, n), row[0].expand(2, 2, n), wide.as_strided((6, n), (1, 1)), row[:, :1].expand(1, n)):
        assert torch.equal(yt.token_probs(t, 0.7), yt.token_probs(t.clone(memory_format=torch.contiguous_format), 0.7))
    one = torch.empty(1, n, device="cuda")
    with pytest.raises(ValueError):
        yt.token_probs(row.expand(4, n).contiguous(), out=one.expand(4, n))
    with pytest.raises(ValueError):
        yt.token_probs(x, out=torch.empty(n + 5, device="cuda").as_strided((3, 1, n), (1, 1, 1)) if n > 1 else one.expand(3, 1, 1))


def test_sizes_past_32_bits():
    """Views of one element with more rows, entries or tokens than 32 bits hold: refused, not taken for their low bits."""
    much, one = (1 << 32) + 5, torch.ones(1, 1, 1, device="cuda")
    for shape in ((much, 1, 1), (1, 1, much), (1 << 16, 1 << 16, 1)):
        with pytest.raises(ValueError, match="2\\^31"):
            yt.token_probs(one.expand(shape))
    zero = torch.zeros(1, 1, device="cuda")
    for B, T, V in ((1, 1, much), (much, 1, 4), (1, much, 4)):
        with pytest.raises(ValueError, match="2\\^31"):
            yt.verify_drafts(one.expand(B, T, V), ints([[0]]).expand(B, T), zero.expand(B, T), zero[0].expand(B))
    pool = torch.zeros(1, 1, 1, yt.cache_q4_bytes(16, 64), dtype=torch.uint8, device="cuda")
    new = torch.zeros(1, 1, 1, 1, 64, device="cuda").expand(1, 1, 1, much, 64)
    with pytest.raises(ValueError, match="2\\^31"):
        yt.cache_append_q4(new, new, pool, pool, ints([[0]]), ints([0]), 16)


@pytest.mark.parametrize("rows,n", [(1, 33), (3, 151936), (200, 33), (200, 80001)])
def test_probs_in_place(rows, n):
    """float32 logits as their own output, in parts and a workgroup a row, and the two halves of one buffer's rows."""
    x = logits((rows, n), torch.float32, n)
    want = yt.token_probs(x, 0.8)
    both = torch.cat([x, torch.zeros_like(x)], 1)
    assert yt.token_probs(both[:, :n], 0.8, out=both[:, n:]).data_ptr() == both.data_ptr() + 4 * n
    assert torch.equal(both[:, n:], want) and torch.equal(both[:, :n], x)
    assert yt.token_probs(both[:, :n], 0.8, out=both[:, :n]).data_ptr() == both.data_ptr()
    assert torch.equal(both[:, :n], want)
    yt.token_probs(x, 0.8, out=x)
    assert torch.equal(x, want)
    if rows > 1:
        with pytest.raises(yt.YthipError):
            yt.token_probs(x[:-1], out=x[1:])


def step(B, T, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    target = torch.softmax(3.0 * torch.randn(B, T, V, generator=g), -1).cuda()
    tokens = torch.multinomial(target.reshape(-1, V).cpu(), 1, generator=g).reshape(B, T).int().cuda()
    return target, tokens, torch.rand(B, T, generator=g).cuda(), torch.rand(B, generator=g).cuda()


def test_outputs_of_a_verification_share_nothing():
    """Outputs over inputs or over each other are refused; those in the gaps of a buffer's rows, and the next token over the
    only one, are as those in memory of their own."""
    B, T, V = 4, 5, 40
    args = step(B, T, V)
    lens = ints([5, 4, 0, 1])
    parents = ints([[0, 0, 1, 1, 2]] * B)
    want = yt.verify_drafts(*args, parents=parents, tree_len=lens)
    ok = lambda: [torch.zeros_like(t) for t in want]  # noqa: E731
    for out in ((args[1], ok()[1], ok()[2]), (parents, ok()[1], ok()[2]), (ok()[0], lens, ok()[2]), (ok()[0], want[1], want[1])):
        with pytest.raises(yt.YthipError):
            yt.verify_drafts(*args, parents=parents, tree_len=lens, out=tuple(out))
    flat = torch.zeros(B * T + 2 * B, dtype=torch.int32, device="cuda")
    out = (flat[: B * T].view(B, T), flat[B * T: B * T + B], flat[B * T + B:])
    yt.verify_drafts(*args, parents=parents, tree_len=lens, out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    # the next token over the only one
    args = step(B, 1, V, 1)
    want = yt.verify_drafts(*args, tree_len=ints([1, 1, 0, 1]))
    out = (torch.zeros_like(want[0]), torch.zeros_like(want[1]), args[1][:, 0])
    yt.verify_drafts(*args, tree_len=ints([1, 1, 0, 1]), out=out)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
