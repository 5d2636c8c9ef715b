"""Sizes past 32 bits, which the C calls cannot be told: refused on the host, never cut to their low bits."""
from __future__ import annotations

import pytest
import torch

import ytensor_amd as yt
from ytensor_amd.paged import _sizes, _table

MUCH = (1 << 32) + 16


def test_a_table_of_too_many_columns():
    assert _table(torch.empty((2, 77), dtype=torch.int32, device="meta"), 2)[1:] == (77, 77)
    with pytest.raises(ValueError, match="2\\^31"):
        _table(torch.empty((1, MUCH), dtype=torch.int32, device="meta"), 1)


def test_pages_of_too_many_rows():
    assert yt.cache_q4_bytes(16, 64) == 16 * 34
    for page, d in ((MUCH, 64), (16, (1 << 32) + 64)):
        with pytest.raises(ValueError):
            yt.cache_q4_bytes(page, d)


def test_sizes_are_handed_on():
    assert _sizes(0, 5, (1 << 31) - 1) == (0, 5, (1 << 31) - 1)
    with pytest.raises(ValueError):
        _sizes(1, 1 << 31)


def test_no_workspace_for_chosen_pages_with_a_window():
    """There is no such attention: the size of one with a window alone is not that of one over chosen pages."""
    args = (torch.bfloat16, 1, 8, 2, 1, 64, 400, 16)
    assert yt.paged_workspace_bytes(*args, top_k=9) > 0 and yt.paged_workspace_bytes(*args, window=99, sinks=3) >= 0
    assert yt.paged_workspace_bytes(*args, top_k=9, sinks=3) == yt.paged_workspace_bytes(*args, top_k=9)
    with pytest.raises(ValueError, match="window"):
        yt.paged_workspace_bytes(*args, top_k=9, window=99)
