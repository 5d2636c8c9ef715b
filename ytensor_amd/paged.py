"""Operators of the paged KV cache over libythip.so (include/ythip.h, "Paged KV cache").

The reference keeps a ring of rows a sequence (KVCache, example/qwen3/src/qwen3.cpp:57-126);
here sequences hold pages of a shared pool, so that they grow without moving, share a
prompt's rows and give them back:

    k_pool, v_pool [P, Hkv, page, d]   (layers in front: [L, P, Hkv, page, d])
    key_sums       [P, Hkv, d] float32 a page's K rows in use added up ([L, P, Hkv, d])
    table          int32 [B, columns]  row r of sequence b: page table[b, r // page], row r % page
    kv_len         int32 [B]           rows in use
    ref            int32 [P]           sequences that hold a page (0: free)

    paged_attention(...)         new tokens (one, a drafted tree, a chunk) over the cache
    paged_sparse_attention(...)  the same over the pages that a score selects
    cache_grow / cache_append    pages for new rows; the rows into them
    cache_fork / cache_free      sequences that share another's pages; their end
    cache_compact / cache_copy_pages

Everything is read on the device when the kernels run, and no call waits for the host, so a
step (attend, keep the lengths, grow in place, append) can be captured as one HIP graph. Argument problems raise
ValueError or YthipError; what only the device can see (no free page, an index out of range)
sets bits of `status`, an int32 device tensor (CACHE_ERR_*).
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._lib import check
from .ops import _DT, _code, _stream

CACHE_ERR_INDEX, CACHE_ERR_BUSY, CACHE_ERR_FULL = 1, 2, 4


@functools.lru_cache(maxsize=4096)
def _i64(vals: tuple) -> ctypes.Array:
    """Strides for the C call, which reads them only (and not the last, of d, nor those of dims of one element)."""
    return _lib.i64array(vals)


def _real(t: torch.Tensor) -> tuple:
    """t's strides, 0 for dims of one element: those may hold anything."""
    return tuple(0 if n == 1 else s for n, s in zip(t.shape, t.stride()))


def _device(first: torch.Tensor, *rest) -> int:
    """The GPU that the tensors (or None) are all on."""
    dev = first.get_device()
    if dev < 0:
        raise ValueError("ytensor_amd operators take device (cuda/hip) tensors")
    for t in rest:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {first.device} and {t.device}")
    return dev


MOST = 2 ** 31 - 1


def _sizes(*sizes: int) -> tuple:
    """The sizes, which the C calls take in 32 bits (asked where there are more than MOST elements: it counts in a call)."""
    if max(sizes) > MOST:
        raise ValueError(f"sizes of {list(sizes)}: 2^31 - 1 at most")
    return sizes


def _away(dev: int):
    """A context that makes `dev` the current GPU, or None where it is that."""
    return None if dev == torch.cuda.current_device() else torch.cuda.device(dev)


def _ints(name: str, t: torch.Tensor, shape: tuple) -> torch.Tensor:
    if t.dtype != torch.int32 or t.shape != shape:
        raise ValueError(f"{name} must be int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t


def _packed(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def _rows(t: torch.Tensor, es: int) -> tuple[torch.Tensor, int, tuple]:
    """t with its last dim contiguous and 16-byte aligned rows (a copy where it has neither), its
    address and strides."""
    at, st = t.data_ptr(), t.stride()
    align = at
    for s in st[:-1]:
        align |= s * es
    if st[-1] != 1 or align & 15:
        align = at
        for s in _real(t)[:-1]:
            align |= s * es
        if st[-1] != 1 or align & 15:
            t = t.clone(memory_format=torch.contiguous_format)
            at, st = t.data_ptr(), t.stride()
    return t, at, st


def _attention(top_k, q, k_new, v_new, k_pool, v_pool, key_sums, table, kv_len, parents, tree_len, scale, out,
               workspace, window=0, sinks=0):
    away = _away(_device(q, k_new, v_new, k_pool, v_pool, key_sums, table, kv_len, parents, tree_len, out, workspace))
    if away is not None:
        with away:
            return _attention(top_k, q, k_new, v_new, k_pool, v_pool, key_sums, table, kv_len, parents, tree_len,
                              scale, out, workspace, window, sinks)
    if q.dim() != 4 or k_pool.dim() != 4:
        raise ValueError("q must be [B, Hq, T, d] and the pools [P, Hkv, page, d]")
    B, Hq, T, d = q.shape
    P, Hkv, page, dk = k_pool.shape
    code, dt = _code(q), q.dtype
    if dk != d or Hkv == 0 or Hq % Hkv != 0:
        raise ValueError(f"q {list(q.shape)} does not fit pools {list(k_pool.shape)}")
    if k_pool.dtype != dt or v_pool.dtype != dt:
        raise ValueError("q and the pools must share a dtype")
    pool_st = k_pool.stride()
    if v_pool.shape != k_pool.shape or pool_st[3] != 1 or (v_pool.stride() != pool_st and _real(v_pool) != _real(k_pool)):
        raise ValueError("k_pool and v_pool must share a shape and strides, with d contiguous")
    es = 4 if dt is torch.float32 else 2
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
    need = _workspace(code, B, Hq, Hkv, T, d, columns, page, top_k or 0, window, sinks)
    ws_at, ws_bytes = None, 0
    if need:
        if workspace is not None and not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        if workspace is None or workspace.numel() * workspace.element_size() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        ws_at, ws_bytes = workspace.data_ptr(), need
    par_at = None if parents is None else parents.data_ptr()
    tl_at = None if tree_len is None else tree_len.data_ptr()
    if top_k is None and window:
        st = _lib.lib().ythip_paged_attn_window(
            code, B, Hq, Hkv, T, d, q_at, _i64(q_st), kn_at, kn_st, vn_at, vn_st, k_pool.data_ptr(),
            v_pool.data_ptr(), _i64(pool_st), P, page, table.data_ptr(), ld, columns, kv_len.data_ptr(), par_at, T,
            tl_at, window, sinks, out.data_ptr(), _i64(out.stride()), scale, ws_at, ws_bytes, _stream())
        if st:
            check(st, "ythip_paged_attn_window")
        return out
    if top_k is None:
        st = _lib.lib().ythip_paged_attn(
            code, B, Hq, Hkv, T, d, q_at, _i64(q_st), kn_at, kn_st, vn_at, vn_st, k_pool.data_ptr(),
            v_pool.data_ptr(), _i64(pool_st), P, page, table.data_ptr(), ld, columns, kv_len.data_ptr(), par_at, T,
            tl_at, out.data_ptr(), _i64(out.stride()), scale, ws_at, ws_bytes, _stream())
        if st:
            check(st, "ythip_paged_attn")
        return out
    if key_sums.dtype != torch.float32 or key_sums.shape != (P, Hkv, d) or key_sums.stride(2) != 1:
        raise ValueError(f"key_sums must be float32 {[P, Hkv, d]} with d contiguous")
    sel = torch.empty((B, Hkv, T, top_k), dtype=torch.int32, device=q.device)
    st = _lib.lib().ythip_paged_attn_sparse(
        code, B, Hq, Hkv, T, d, q_at, _i64(q_st), kn_at, kn_st, vn_at, vn_st, k_pool.data_ptr(),
        v_pool.data_ptr(), _i64(pool_st), P, page, key_sums.data_ptr(), _i64(key_sums.stride()),
        table.data_ptr(), ld, columns, kv_len.data_ptr(), par_at, T, tl_at, top_k, sel.data_ptr(), out.data_ptr(),
        _i64(out.stride()), scale, ws_at, ws_bytes, _stream())
    if st:
        check(st, "ythip_paged_attn_sparse")
    return out, sel


def _table(table: torch.Tensor, B: int) -> tuple[torch.Tensor, int, int]:
    """(table, row stride, columns)"""
    if table.dim() != 2:
        raise ValueError("table must be int32 [B, columns]")
    columns = table.shape[1]
    if table.numel() > MOST:
        _sizes(*table.shape)
    _ints("table", table, (B, columns))
    ld, step = table.stride()
    if step != 1 and columns > 1:
        raise ValueError("table must have contiguous rows")
    return table, ld if B > 1 else max(ld, columns), columns  # a single row has no stride


@functools.lru_cache(maxsize=4096)
def _workspace(code, B, Hq, Hkv, T, d, columns, page, top_k, window=0, sinks=0) -> int:
    if window:
        return int(_lib.lib().ythip_paged_attn_window_workspace_size(code, B, Hq, Hkv, T, d, columns, page, window, sinks))
    if top_k:
        return int(_lib.lib().ythip_paged_attn_sparse_workspace_size(code, B, Hq, Hkv, T, d, columns, page, top_k))
    return int(_lib.lib().ythip_paged_attn_workspace_size(code, B, Hq, Hkv, T, d, columns, page))


def paged_workspace_bytes(dtype: torch.dtype, B: int, Hq: int, Hkv: int, T: int, d: int, columns: int, page: int,
                          top_k: int = 0, window: int = 0, sinks: int = 0) -> int:
    """Bytes that paged_attention (top_k 0) or paged_sparse_attention, which has no window, writes."""
    if top_k and window:
        raise ValueError(f"top_k = {top_k} and a window of {window}: attention over chosen pages has no window")
    return _workspace(_DT[dtype], B, Hq, Hkv, T, d, columns, page, top_k, *_window(window, sinks))


def _window(window, sinks) -> tuple[int, int]:
    """The window as the C calls take it."""
    if window < 0 or sinks < 0:
        raise ValueError(f"a window of {window} and {sinks} sinks")
    return (min(int(window), 2 ** 31 - 1), min(int(sinks), 2 ** 31 - 1)) if window else (0, 0)


def paged_attention(q: torch.Tensor, k_new: torch.Tensor | None, v_new: torch.Tensor | None, k_pool: torch.Tensor,
                    v_pool: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor,
                    parents: torch.Tensor | None = None, tree_len: torch.Tensor | None = None, scale: float = 0.0,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, window: int = 0,
                    sinks: int = 0) -> torch.Tensor:
    """Attention of T new tokens a sequence, q [B, Hq, T, d], over the kv_len[b] cached rows of
    a layer's pools and the tokens' own k_new / v_new [B, Hkv, T, d] (None: the cache alone).

    parents int32 [B, T]: the new tokens are a drafted tree, token t sees itself, parents[b, t],
    that one's parent, ... up to a value outside [0, child) (the cache's last row). None: token t
    sees the new tokens 0..t (T = 1: a decode step; a chunk of a prompt). tree_len int32 [B]: the
    new tokens of each sequence; rows behind them in `out` are left as they were (zeros in an
    `out` made here). Query head h reads KV head h // (Hq // Hkv). A page id outside the pool
    hides its rows; a row that sees nothing is zero. d 64 or 128, page a power of two >= 16.
    window > 0: of these, a token sees what lies less than `window` positions before it (itself the first), and the
    first `sinks` positions. Cached row r is at position r, new token t at kv_len[b] + the tokens above it.
    Returns out [B, Hq, T, d]."""
    return _attention(None, q, k_new, v_new, k_pool, v_pool, None, table, kv_len, parents, tree_len, float(scale), out,
                      workspace, *_window(window, sinks))


def paged_sparse_attention(q: torch.Tensor, k_new: torch.Tensor | None, v_new: torch.Tensor | None,
                           k_pool: torch.Tensor, v_pool: torch.Tensor, key_sums: torch.Tensor, table: torch.Tensor,
                           kv_len: torch.Tensor, top_k: int, parents: torch.Tensor | None = None,
                           tree_len: torch.Tensor | None = None, scale: float = 0.0,
                           out: torch.Tensor | None = None,
                           workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """paged_attention over top_k of the sequence's pages, chosen for each new token and KV head:
    the last page, then those with the highest (sum of the token's queries of that KV head) .
    key_sums[page] (in 64 bits; equal ones and NaN, the lowest, by the lower index). key_sums as
    cache_append keeps them. Returns (out, sel): sel int32 [B, Hkv, T, top_k] holds the chosen
    table columns ascending, then -1 (-1 alone for t >= tree_len[b])."""
    if top_k < 1:
        raise ValueError(f"top_k = {top_k}: at least one page")
    return _attention(int(top_k), q, k_new, v_new, k_pool, v_pool, key_sums, table, kv_len, parents, tree_len,
                      float(scale), out, workspace)


# ---------------------------------------------------------------------------
# The cache's rows and pages
# ---------------------------------------------------------------------------

def _state(ref, table, kv_len, out, page, status):
    """(arguments up to len, arguments of the outputs, the outputs) of a bookkeeping call."""
    if table.dim() != 2 or ref.dim() != 1:
        raise ValueError("table must be int32 [B, columns] and ref int32 [P]")
    B, pages = table.shape[0], ref.shape
    out = (ref, table, kv_len) if out is None else tuple(out)
    args = []
    for r, t, n in ((ref, table, kv_len), out):
        t, ld, columns = _table(t, B)
        if columns != table.shape[1]:
            raise ValueError("the tables must have the same columns")
        if not _ints("ref", r, pages).is_contiguous() or not _ints("kv_len", n, (B,)).is_contiguous():
            raise ValueError("ref and kv_len must be contiguous")
        args.append((r.data_ptr(), t.data_ptr(), ld, n.data_ptr()))
    if status is not None:
        _ints("status", status, (1,))
    return (B, table.shape[1], pages[0], page, *args[0]), args[1], out


def _list(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int32 or t.dim() != 1:
        raise ValueError(f"{name} must be int32 [n]")
    return _packed(t)


@functools.lru_cache(maxsize=4096)
def _pool_layout(shape: tuple, stride: tuple, es: int) -> tuple:
    """(layers, pages, layer stride, page stride, page bytes) of a [L, P, ...] tensor, in bytes."""
    if len(shape) < 3:
        raise ValueError(f"a pool of shape {list(shape)}; needs [layers, pages, ...]")
    inner = 1
    for size, step in zip(reversed(shape[2:]), reversed(stride[2:])):
        if size != 1 and step != inner:
            raise ValueError(f"a pool of shape {list(shape)} and strides {list(stride)}: a page must be contiguous")
        inner *= size
    layer, page = (0 if n == 1 else step * es for n, step in zip(shape[:2], stride[:2]))
    return shape[0], shape[1], layer, page, inner * es


def _pools(pools, pages: int):
    """(pools, layers, their ythip_page_pool descriptors)"""
    layers, words = None, []
    for t in pools:
        n, p, ls, ps, size = _pool_layout(t.shape, t.stride(), t.element_size())
        if p != pages or (layers is not None and n != layers):
            raise ValueError(f"a pool of shape {list(t.shape)}; needs [{'layers' if layers is None else layers}, {pages}, ...]")
        layers = n
        words += (t.data_ptr(), ls, ps, size)
    return len(pools), layers or 0, (ctypes.c_int64 * len(words))(*words)


def cache_grow(ref: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, n_new: torch.Tensor, page: int,
               out=None, status: torch.Tensor | None = None):
    """Pages (lowest free first) for n_new[b] more rows of each sequence, and the new lengths.
    A sequence that finds too few pages or columns keeps what it has (status). out: (ref,
    table, kv_len) to write instead of the given ones. Returns those written. cache_append
    takes the kv_len from before and these new ones."""
    away = _away(_device(ref, table, kv_len, n_new, status, *(out or ())))
    if away is not None:
        with away:
            return cache_grow(ref, table, kv_len, n_new, page, out, status)
    head, tail, out = _state(ref, table, kv_len, out, page, status)
    n_new = _packed(_ints("n_new", n_new, (head[0],)))
    st = _lib.lib().ythip_cache_grow(*head, n_new.data_ptr(), *tail, None if status is None else status.data_ptr(),
                                     _stream())
    if st:
        check(st, "ythip_cache_grow")
    return out


def cache_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 table: torch.Tensor, kv_len: torch.Tensor, n_new: torch.Tensor | None = None,
                 path: torch.Tensor | None = None, key_sums: torch.Tensor | None = None,
                 new_len: torch.Tensor | None = None, status: torch.Tensor | None = None) -> None:
    """Cached row kv_len[b] + i of sequence b takes row path[b, i] (None: i) of k_new / v_new
    [L, B, Hkv, T, d], for every layer; pools [L, P, Hkv, page, d]. A path entry outside [0, T)
    writes zeros. key_sums [L, P, Hkv, d]: the sums of the pages written to.

    kv_len is the length before, table holds the pages already (cache_grow). new_len: the
    lengths that cache_grow wrote, in a tensor of their own; a sequence that it refused gets no row, rows past the T given
    are zeros, and lengths or page ids that cannot be set CACHE_ERR_INDEX in `status`. Without
    new_len i < n_new[b] (None: T), each of which must have its page in the table."""
    away = _away(_device(k_new, v_new, k_pool, v_pool, table, kv_len, n_new, path, key_sums, new_len, status))
    if away is not None:
        with away:
            return cache_append(k_new, v_new, k_pool, v_pool, table, kv_len, n_new, path, key_sums, new_len, status)
    if new_len is None and status is not None:
        raise ValueError("status goes with new_len")
    if new_len is not None and n_new is not None:
        raise ValueError("n_new and new_len both say how many rows there are: give one")
    if k_new.dim() != 5 or k_pool.dim() != 5:
        raise ValueError("k_new must be [L, B, Hkv, T, d] and the pools [L, P, Hkv, page, d]")
    L, B, Hkv, T, d = k_new.shape
    P, page = k_pool.shape[1], k_pool.shape[3]
    if tuple(k_pool.shape) != (L, P, Hkv, page, d) or k_pool.shape != v_pool.shape or k_new.shape != v_new.shape:
        raise ValueError(f"k_new {list(k_new.shape)}, v_new {list(v_new.shape)}, pools {list(k_pool.shape)}, "
                         f"{list(v_pool.shape)} do not fit")
    if not (k_new.dtype == v_new.dtype == k_pool.dtype == v_pool.dtype):
        raise ValueError("k_new, v_new and the pools must share a dtype")
    if k_pool.stride(4) != 1 or (k_pool.stride() != v_pool.stride() and _real(k_pool) != _real(v_pool)):
        raise ValueError("k_pool and v_pool must share strides, with d contiguous")
    es = k_new.element_size()
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
    if key_sums is not None and (key_sums.dtype != torch.float32 or key_sums.shape != (L, P, Hkv, d)
                                 or key_sums.stride(3) != 1):
        raise ValueError(f"key_sums must be float32 {[L, P, Hkv, d]} with d contiguous")
    head = (_code(k_new), L, B, Hkv, T, d, k_at, v_at, _i64(new_st), k_pool.data_ptr(), v_pool.data_ptr(),
            _i64(k_pool.stride()), P, page, None if key_sums is None else key_sums.data_ptr(),
            None if key_sums is None else _i64(key_sums.stride()), table.data_ptr(), ld, columns, kv_len.data_ptr())
    path_at = None if path is None else path.data_ptr()
    if new_len is None:
        st = _lib.lib().ythip_cache_append(*head, None if n_new is None else n_new.data_ptr(), path_at, T, _stream())
        if st:
            check(st, "ythip_cache_append")
        return
    st = _lib.lib().ythip_cache_append_to(*head, new_len.data_ptr(), path_at, T,
                                          None if status is None else status.data_ptr(), _stream())
    if st:
        check(st, "ythip_cache_append_to")


def cache_fork(pools, ref: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, src: torch.Tensor,
               dst: torch.Tensor, page: int, out=None, status: torch.Tensor | None = None):
    """Sequence dst[i] (empty before) becomes a copy of src[i]: it shares the whole pages and
    gets a copy of the partial last one, in every pool ([L, P, ...] tensors: K, V, key sums).
    All pairs read the state before the call. A pair that is refused (dst in use or named
    twice, no free page, an index out of range) leaves dst empty (status). out and the result
    as for cache_grow."""
    away = _away(_device(ref, table, kv_len, src, dst, status, *pools, *(out or ())))
    if away is not None:
        with away:
            return cache_fork(pools, ref, table, kv_len, src, dst, page, out, status)
    head, tail, out = _state(ref, table, kv_len, out, page, status)
    src, dst = _list("src", src), _list("dst", dst)
    if src.shape != dst.shape:
        raise ValueError("src and dst must have the same length")
    n = src.shape[0]
    n_pools, layers, descr = _pools(pools, ref.shape[0])
    ws = torch.empty(max(int(_lib.lib().ythip_cache_fork_workspace_size(n)), 16), dtype=torch.uint8, device=ref.device)
    check(_lib.lib().ythip_cache_fork(*head, n, src.data_ptr(), dst.data_ptr(), *tail, n_pools, layers, descr,
                                      None if status is None else status.data_ptr(), ws.data_ptr(), ws.numel(),
                                      _stream()), "ythip_cache_fork")
    return out


def cache_free(ref: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, seqs: torch.Tensor, page: int, out=None,
               status: torch.Tensor | None = None):
    """The pages of sequences seqs lose a user; their table rows become -1, their lengths 0.
    An empty sequence and a second mention change nothing. out and the result as for cache_grow."""
    away = _away(_device(ref, table, kv_len, seqs, status, *(out or ())))
    if away is not None:
        with away:
            return cache_free(ref, table, kv_len, seqs, page, out, status)
    head, tail, out = _state(ref, table, kv_len, out, page, status)
    seqs = _list("seqs", seqs)
    check(_lib.lib().ythip_cache_free(*head, seqs.shape[0], seqs.data_ptr(), *tail,
                                      None if status is None else status.data_ptr(), _stream()), "ythip_cache_free")
    return out


def cache_compact(pools, ref: torch.Tensor, table: torch.Tensor, kv_len: torch.Tensor, page: int, out=None):
    """Moves the pages in use to the front of every pool ([L, P, ...] tensors), in order, and
    has ref and table follow. out: (ref, table) to write instead of the given ones. Returns
    (ref, table, live): live int32 [1], the pages in use."""
    away = _away(_device(ref, table, kv_len, *pools, *(out or ())))
    if away is not None:
        with away:
            return cache_compact(pools, ref, table, kv_len, page, out)
    out = (ref, table) if out is None else tuple(out)
    head, tail, out = _state(ref, table, kv_len, (*out, kv_len), page, None)
    n_pools, layers, descr = _pools(pools, ref.shape[0])
    live = torch.empty(1, dtype=torch.int32, device=ref.device)
    ws = torch.empty(int(_lib.lib().ythip_cache_compact_workspace_size(ref.shape[0])), dtype=torch.uint8,
                     device=ref.device)
    check(_lib.lib().ythip_cache_compact(*head, *tail[:3], live.data_ptr(), n_pools, layers, descr, ws.data_ptr(),
                                         ws.numel(), _stream()), "ythip_cache_compact")
    return out[0], out[1], live


def cache_copy_pages(pools, src: torch.Tensor, dst: torch.Tensor, status: torch.Tensor | None = None) -> None:
    """Page src[i] over page dst[i] of every pool ([L, P, ...] tensors). No dst may be another
    pair's src or dst; a pair with an index out of range is left out (status)."""
    away = _away(_device(src, dst, status, *pools))
    if away is not None:
        with away:
            return cache_copy_pages(pools, src, dst, status)
    src, dst = _list("src", src), _list("dst", dst)
    if src.shape != dst.shape:
        raise ValueError("src and dst must have the same length")
    if len(pools) == 0:
        return
    if status is not None:
        _ints("status", status, (1,))
    pages = pools[0].shape[1] if pools[0].dim() >= 3 else 0
    n_pools, layers, descr = _pools(pools, pages)
    check(_lib.lib().ythip_cache_copy_pages(pages, src.shape[0], src.data_ptr(), dst.data_ptr(), n_pools, layers,
                                            descr, None if status is None else status.data_ptr(), _stream()),
          "ythip_cache_copy_pages")
