"""4-bit pools of many GB on the GPU: offsets past 32 bits and more workgroups than one launch holds."""
from __future__ import annotations

import pytest
import torch

import q4_ref
import ytensor_amd as yt

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_behind_4_gb(dtype):
    """Rows into the last pages of a pool of 5 GB and attention over them: the bits that a pool of these pages alone gives."""
    page, d, Hkv, P, B, T = 64, 128, 8, 150000, 3, 40
    g = torch.Generator().manual_seed(1)
    size = yt.cache_q4_bytes(page, d)
    k, v = (torch.empty(1, P, Hkv, size, dtype=torch.uint8, device="cuda") for _ in range(2))
    assert (P - 1) * Hkv * size > 1 << 32
    small = [torch.randint(100, 140, (1, 9, Hkv, size), generator=g).to(torch.uint8).cuda() for _ in range(2)]
    for big, part in zip((k, v), small):
        big[:, P - 9:] = part
    new = [torch.randn(1, B, Hkv, T, d, generator=g).to(dtype).cuda() for _ in range(3)]
    table, kv_len = ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]]), ints([100, 64, 37])
    q = new[2][0].repeat_interleave(2, 1)
    outs = []
    for pools, first in (((k, v), P - 9), (small, 0)):
        yt.cache_append_q4(new[0], new[1], *pools, table + first, kv_len, page)
        outs.append(yt.paged_attention_q4(q, new[0][0], new[1][0], pools[0][0], pools[1][0], table + first, kv_len + T, page))
    assert all(torch.equal(big[:, P - 9:], part) for big, part in zip((k, v), small))
    assert torch.isfinite(outs[0]).all() and torch.equal(*outs)


@pytest.mark.parametrize("d", [64, 128])
def test_values_of_a_large_pool(d):
    """The values of all pages of two layers, 4 GB of blocks: a few blocks from the start, the end and around every 2^23rd
    group of 16 rows."""
    L, Hkv, page = 2, 8, 128
    P = 34000 * 64 // d * 2
    size = yt.cache_q4_bytes(page, d)
    blocks = L * P * Hkv
    assert 2 * blocks * (page // 16) > 1 << 23
    k, v = (torch.randint(100, 140, (L, P, Hkv, size), dtype=torch.uint8, device="cuda") for _ in range(2))
    out = yt.cache_unpack_q4(k, v, page, torch.bfloat16)
    cut = (1 << 23) // (2 * (page // 16))
    for b in (0, 1, blocks // 2, blocks - 1, *(x for c in range(cut, blocks, cut) for x in (c - 1, c))):
        for pool, values, which in ((k, out[0], "k"), (v, out[1], "v")):
            want = q4_ref.values(pool.view(blocks, size)[b], page, d, which).to(torch.bfloat16)
            assert torch.equal(values.view(blocks, page, d)[b].cpu(), want), (b, which)
