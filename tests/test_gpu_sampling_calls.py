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
