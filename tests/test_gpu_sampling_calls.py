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
