"""The paged KV cache in 4 bits over libythip.so (include/ythip.h, "4-bit pages"): a quarter of the 16-bit cache's bytes
and a little for the scales.

    k_pool, v_pool uint8 [P, Hkv, cache_q4_bytes(page, d)]   (layers in front: [L, P, Hkv, ...])

A page and KV head is a block: the codes of its rows, then their scales. Groups of 32 neighbouring channels of a row share
a scale, a power of two (a byte, its exponent + 127; 255: the group has no value); a code is a sign (8) and one of 0, 0.5,
1, 1.5, 2, 3, 4, 6 (0 to 7), channel 2 i in the low half of its byte:

    K   codes [page][d / 2], scales [page][d / 32]
    V   codes [page / 8][16][8][d / 32], entry i of 16: channels i d / 16 and on of 8 rows; scales [page / 8][d / 32][8]

The table, the lengths and the bookkeeping are those of the paged cache (ytensor_amd/paged.py): cache_grow, cache_fork,
cache_free and cache_compact take these pools as they are.

    cache_append_q4(...)      the new tokens' rows of every layer into the pages
    cache_unpack_q4(...)      the values that the pages hold
    paged_attention_q4(...)   new tokens (one, a drafted tree, a chunk) over the cache
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from ._lib import check
from .ops import _DT, _code, _stream
from .paged import MOST, _away, _device, _i64, _ints, _packed, _real, _rows, _sizes, _table, _window


@functools.lru_cache(maxsize=256)
def cache_q4_bytes(page: int, d: int) -> int:
    """Bytes of a page and KV head: page (d / 2 + d / 32)."""
    n = int(_lib.lib().ythip_cache_q4_bytes(*_sizes(page, d)))
    if n == 0:
        raise ValueError(f"a page of {page} rows of {d}: needs a power of two from 16 to 32768 and a head dim of 64 or 128")
    return n


def _blocks(k_pool: torch.Tensor, v_pool: torch.Tensor, dims: int) -> tuple:
    """The strides that the pools share."""
    if k_pool.dtype != torch.uint8 or v_pool.dtype != torch.uint8 or k_pool.dim() != dims or v_pool.shape != k_pool.shape:
        raise ValueError(f"4-bit pools must be uint8 [{'L, ' if dims == 4 else ''}P, Hkv, bytes], got {k_pool.dtype} "
                         f"{list(k_pool.shape)} and {v_pool.dtype} {list(v_pool.shape)}")
    st = k_pool.stride()
    if st[-1] != 1 or (v_pool.stride() != st and (v_pool.stride(-1) != 1 or _real(v_pool) != _real(k_pool))):
        raise ValueError("k_pool and v_pool must share strides, with a block contiguous")
    return st


def _head_dim(pool: torch.Tensor, page: int) -> int:
    for d in (64, 128):
        if pool.shape[-1] == cache_q4_bytes(page, d):
            return d
    raise ValueError(f"blocks of {pool.shape[-1]} bytes are not those of pages of {page} rows")


def cache_append_q4(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                    table: torch.Tensor, kv_len: torch.Tensor, page: int, n_new: torch.Tensor | None = None,
                    path: torch.Tensor | None = None, new_len: torch.Tensor | None = None,
                    status: torch.Tensor | None = None) -> None:
    """cache_append into 4-bit pools [L, P, Hkv, cache_q4_bytes(page, d)]: cached row kv_len[b] + i of sequence b takes row
    path[b, i] (None: i) of k_new / v_new [L, B, Hkv, T, d]. kv_len, table, path, n_new, new_len and status as there.

    A group's scale is the smallest power of two with which its largest magnitude is at most 7, so that no value is
    further off than half a step; a value takes the nearest code, of two as near the even one. The scale is at least 2^-125
    and at most 2^125 (float16: 2^13), so that every value is one of the type's; what lies beyond 6 times that takes it.
    A group with a NaN or an infinity has no value (scale byte 255: it reads as NaN)."""
    away = _away(_device(k_new, v_new, k_pool, v_pool, table, kv_len, n_new, path, new_len, status))
    if away is not None:
        with away:
            return cache_append_q4(k_new, v_new, k_pool, v_pool, table, kv_len, page, n_new, path, new_len, status)
    if new_len is None and status is not None:
        raise ValueError("status goes with new_len")
    if new_len is not None and n_new is not None:
        raise ValueError("n_new and new_len both say how many rows there are: give one")
    if k_new.dim() != 5:
        raise ValueError("k_new must be [L, B, Hkv, T, d]")
    L, B, Hkv, T, d = k_new.shape
    if k_new.numel() > MOST:
        _sizes(*k_new.shape)
    pool_st = _blocks(k_pool, v_pool, 4)
    P = k_pool.shape[1]
    if tuple(k_pool.shape) != (L, P, Hkv, cache_q4_bytes(page, d)) or v_new.shape != k_new.shape or v_new.dtype != k_new.dtype:
        raise ValueError(f"k_new {list(k_new.shape)}, v_new {list(v_new.shape)} and pools {list(k_pool.shape)} of pages of "
                         f"{page} rows do not fit")
    es = k_new.element_size()
    code = _code(k_new)
    k_new, k_at, new_st = _rows(k_new, es)
    v_new, v_at, v_st = _rows(v_new, es)
    if new_st != v_st and _real(k_new) != _real(v_new):
        k_new, v_new = (t.clone(memory_format=torch.contiguous_format) for t in (k_new, v_new))
        k_at, v_at, new_st = k_new.data_ptr(), v_new.data_ptr(), k_new.stride()
    table, ld, columns = _table(table, B)
    kv_len = _packed(_ints("kv_len", kv_len, (B,)))
    if n_new is not None:
        n_new = _packed(_ints("n_new", n_new, (B,)))
    if new_len is not None:
        new_len = _packed(_ints("new_len", new_len, (B,)))
    if status is not None:
        _ints("status", status, (1,))
    if path is not None:
        path = _packed(_ints("path", path, (B, T)))
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    st = _lib.lib().ythip_cache_append_q4(code, L, B, Hkv, T, d, k_at, v_at, _i64(new_st), k_pool.data_ptr(), v_pool.data_ptr(),
                                          _i64(pool_st), P, page, table.data_ptr(), ld, columns, kv_len.data_ptr(), at(n_new),
                                          at(new_len), at(path), T, at(status), _stream())
    if st:
        check(st, "ythip_cache_append_q4")


def cache_unpack_q4(k_pool: torch.Tensor, v_pool: torch.Tensor, page: int, dtype: torch.dtype = torch.float32,
                    out=None) -> tuple[torch.Tensor, torch.Tensor]:
    """What 4-bit pools [L, P, Hkv, bytes] hold, as K and V [L, P, Hkv, page, d] of `dtype` (out: two such contiguous
    tensors to write, in memory of their own), whatever their rows are in use for. Values that the type cannot hold are rounded to it."""
    away = _away(_device(k_pool, v_pool, *(out or ())))
    if away is not None:
        with away:
            return cache_unpack_q4(k_pool, v_pool, page, dtype, out)
    st = _blocks(k_pool, v_pool, 4)
    d = _head_dim(k_pool, page)
    if dtype not in _DT:
        raise ValueError(f"unsupported dtype {dtype}")
    L, P, Hkv, _ = k_pool.shape
    shape = (L, P, Hkv, page, d)
    if out is None:
        out = tuple(torch.empty(shape, dtype=dtype, device=k_pool.device) for _ in range(2))
    k, v = out
    for t in (k, v):
        if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"out must be two contiguous {dtype} {list(shape)}")
    check(_lib.lib().ythip_cache_unpack_q4(_DT[dtype], L, P, Hkv, page, d, k_pool.data_ptr(), v_pool.data_ptr(), _i64(st),
                                           k.data_ptr(), v.data_ptr(), _stream()), "ythip_cache_unpack_q4")
    return k, v


@functools.lru_cache(maxsize=4096)
def _workspace_q4(code, B, Hq, Hkv, T, d, columns, page, window, sinks) -> int:
    return int(_lib.lib().ythip_paged_attn_q4_workspace_size(code, B, Hq, Hkv, T, d, columns, page, window, sinks))


def paged_q4_workspace_bytes(dtype: torch.dtype, B: int, Hq: int, Hkv: int, T: int, d: int, columns: int, page: int,
                             window: int = 0, sinks: int = 0) -> int:
    """Bytes that paged_attention_q4 writes."""
    return _workspace_q4(_DT[dtype], B, Hq, Hkv, T, d, columns, page, *_window(window, sinks))


def paged_attention_q4(q: torch.Tensor, k_new: torch.Tensor | None, v_new: torch.Tensor | None, k_pool: torch.Tensor,
                       v_pool: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, page: int,
                       parents: torch.Tensor | None = None, tree_len: torch.Tensor | None = None, scale: float = 0.0,
                       out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, window: int = 0,
                       sinks: int = 0) -> torch.Tensor:
    """paged_attention over a layer's 4-bit pools [P, Hkv, cache_q4_bytes(page, d)]: T new tokens a sequence, q [B, Hq, T,
    d] of any of the three types, over the kv_len[b] cached rows' values and the tokens' own k_new / v_new [B, Hkv, T, d] of
    q's type (None: the cache alone). parents, tree_len, scale, out, window and sinks as there. The cached values take part
    as they are, whatever q's type is. An infinity or a NaN in a query has the scores that follow from it: -inf has no
    weight (a row that has nothing else is zero), +inf and NaN make the row NaN. Returns out [B, Hq, T, d]."""
    away = _away(_device(q, k_new, v_new, k_pool, v_pool, table, kv_len, parents, tree_len, out, workspace))
    if away is not None:
        with away:
            return paged_attention_q4(q, k_new, v_new, k_pool, v_pool, table, kv_len, page, parents, tree_len, scale, out,
                                      workspace, window, sinks)
    if q.dim() != 4:
        raise ValueError("q must be [B, Hq, T, d]")
    B, Hq, T, d = q.shape
    code, dt = _code(q), q.dtype
    pool_st = _blocks(k_pool, v_pool, 3)
    P, Hkv, size = k_pool.shape
    if size != cache_q4_bytes(page, d) or Hkv == 0 or Hq % Hkv != 0:
        raise ValueError(f"q {list(q.shape)} does not fit 4-bit pools {list(k_pool.shape)} of pages of {page} rows")
    es = q.element_size()
    q, q_at, q_st = _rows(q, es)
    kn_at = vn_at = kn_st = vn_st = None
    if k_new is not None and v_new is not None:
        want = (B, Hkv, T, d)
        if k_new.shape != want or v_new.shape != want or k_new.dtype != dt or v_new.dtype != dt:
            raise ValueError(f"k_new and v_new must be {dt} {list(want)}")
        k_new, kn_at, kn_st = _rows(k_new, es)
        v_new, vn_at, vn_st = _rows(v_new, es)
        kn_st, vn_st = _i64(kn_st), _i64(vn_st)
    elif k_new is not None or v_new is not None:
        raise ValueError("k_new and v_new go together")
    table, ld, columns = _table(table, B)
    kv_len = _packed(_ints("kv_len", kv_len, (B,)))
    if parents is not None:
        parents = _packed(_ints("parents", parents, (B, T)))
    if tree_len is not None:
        tree_len = _packed(_ints("tree_len", tree_len, (B,)))
    if out is None:
        out = (torch.empty if tree_len is None else torch.zeros)((B, Hq, T, d), dtype=dt, device=q.device)
    elif out.shape != (B, Hq, T, d) or out.dtype != dt or out.stride(3) != 1:
        raise ValueError(f"out must be {dt} {[B, Hq, T, d]} with d contiguous")
    window, sinks = _window(window, sinks)
    need = _workspace_q4(code, B, Hq, Hkv, T, d, columns, page, window, sinks)
    ws_at, ws_bytes = None, 0
    if need:
        if workspace is not None and not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        if workspace is None or workspace.numel() * workspace.element_size() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        ws_at, ws_bytes = workspace.data_ptr(), need
    st = _lib.lib().ythip_paged_attn_q4(
        code, B, Hq, Hkv, T, d, q_at, _i64(q_st), kn_at, kn_st, vn_at, vn_st, k_pool.data_ptr(), v_pool.data_ptr(),
        _i64(pool_st), P, page, table.data_ptr(), ld, columns, kv_len.data_ptr(), None if parents is None else parents.data_ptr(),
        T, None if tree_len is None else tree_len.data_ptr(), window, sinks, out.data_ptr(), _i64(out.stride()), float(scale),
        ws_at, ws_bytes, _stream())
    if st:
        check(st, "ythip_paged_attn_q4")
    return out
