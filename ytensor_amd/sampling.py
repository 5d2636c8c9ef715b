"""The end of a drafted step over libythip.so (include/ythip.h, "Drafted tokens"): probabilities from logits, and the
drafted tokens that are kept. The reference's step ends with the greedy token (example/qwen3/src/qwen3.cpp:465-486;
argmax_step here).

    p = token_probs(logits, temperature)               # of the target's T new tokens a sequence
    path, kept, token = verify_drafts(p, tokens, u, u_next, parents=parents, tree_len=tree_len)
    # path and kept are what cache_grow and cache_append take; `token` opens the next step

Nothing waits for the host, so a step can be captured as one HIP graph.
"""
from __future__ import annotations

import functools

import torch

from . import _lib
from ._lib import check
from .ops import _code, _stream
from .paged import MOST, _away, _device, _i64, _ints, _packed, _sizes


def token_probs(logits: torch.Tensor, temperature: float = 1.0, out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(logits / temperature) over the last dim, in float32 (out: float32 of logits' shape). A logit of -inf has
    probability 0, a row of them zeros; a NaN or +inf makes its row NaN. temperature > 0. out may be float32 logits
    themselves, else it shares no memory with them."""
    away = _away(_device(logits, out, workspace))
    if away is not None:
        with away:
            return token_probs(logits, temperature, out, workspace)
    code, shape = _code(logits), logits.shape
    if logits.dim() < 1:
        raise ValueError("logits must be [..., V]")
    if logits.numel() > MOST:
        _sizes(logits.numel() // shape[-1], shape[-1])
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=logits.device)
    elif out.dtype != torch.float32 or out.shape != shape:
        raise ValueError(f"out must be float32 {list(shape)}")
    n = shape[-1]
    if logits.is_contiguous() and out.is_contiguous() and n:
        x, o, rows, ld, ld_out = logits, out, logits.numel() // n, n, n
    else:
        x, o, rows, ld, ld_out = _matrices(logits, out, n)
    at, size, need = None, 0, _probs_workspace(rows, n)
    if need:
        workspace, at, size = _space(workspace, need, logits.device)
    st = _lib.lib().ythip_token_probs(code, rows, n, x.data_ptr(), ld, float(temperature), o.data_ptr(), ld_out, at, size,
                                      _stream())
    if st:
        check(st, "ythip_token_probs")
    return out


def _matrices(logits, out, n):
    """logits and out as rows: (logits, or a copy, out, rows, their strides)"""
    x, o = _matrix(logits), _matrix(out)
    if x is None:
        x = logits.contiguous().reshape(-1, n)
    if o is None:
        raise ValueError("out must have rows at one stride, with the last dim contiguous")
    return x, o, x.shape[0], x.stride(0), o.stride(0)


def _matrix(t: torch.Tensor) -> torch.Tensor | None:
    """t as [rows, n] without a copy; None where its rows do not lie at one stride, one behind the other, or its last dim is
    not contiguous."""
    n = t.shape[-1]
    if n > 1 and t.stride(-1) != 1:
        return None
    if t.numel() == 0:
        return t.new_empty((0, n))
    try:
        m = t.view(-1, n)
    except RuntimeError:
        return None
    return m if m.shape[0] == 1 or m.stride(0) >= n else None


@functools.lru_cache(maxsize=4096)
def _probs_workspace(rows: int, n: int) -> int:
    return int(_lib.lib().ythip_token_probs_workspace_size(rows, n))


@functools.lru_cache(maxsize=4096)
def _verify_workspace(B: int, V: int) -> int:
    return int(_lib.lib().ythip_verify_drafts_workspace_size(B, V))


def _space(workspace, need: int, device):
    """(workspace, its address, bytes): the given one, or one made here, of `need` bytes."""
    if need == 0:
        return None, None, 0
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    return workspace, workspace.data_ptr(), need


def _floats(name: str, t: torch.Tensor, shape: tuple) -> torch.Tensor:
    if t.dtype != torch.float32 or t.shape != shape:
        raise ValueError(f"{name} must be float32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return _packed(t)


def verify_drafts(target: torch.Tensor, tokens: torch.Tensor, u: torch.Tensor, u_next: torch.Tensor,
                  draft: torch.Tensor | None = None, parents: torch.Tensor | None = None,
                  tree_len: torch.Tensor | None = None, out=None,
                  workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which of a sequence's new tokens are kept, so that what is kept and the token after it are distributed as the
    target's, and that next token, from given random numbers in [0, 1).

    target [B, T, V]: the target's probabilities after each new token (token_probs; any of the three types). tokens int32
    [B, T]: the new tokens; token 0 is known and always kept. parents int32 [B, T] as in paged_attention (None: a chain,
    each after the one before it); tree_len int32 [B]: the new tokens of each sequence.

    Without draft: from token n, u[b, n] falls into one of the intervals that its children's probabilities, in the order
    of the children, take of [0, 1) (the first of several with one token has it), and that child is kept, or into none;
    the next token is then drawn by u_next[b] from n's row without its children's tokens. With draft [B, T, V], the
    probabilities that token t was drawn from (a chain: no parents): t is kept while u[b, t] draft[b, t, token] <
    target[b, t - 1, token]; the next token is drawn from the row of the last kept one less draft's row of the refused
    one, where that is positive. After the last of a path nothing is taken off. Where nothing is left the row is taken
    as it is. A draw is the first entry at which the sum passes u_next[b] times all; what is not a positive number has
    no weight. Decided in 64 bits.

    Returns (path, kept, token), int32 [B, T], [B], [B]: the kept tokens' numbers, then -1; how many; the next token (-1
    where tree_len is 0 or the row has no weight). out: three such tensors to write, in memory of their own (the last may
    be the tokens where T is 1). At most 1024 tokens a sequence and 2^22 entries."""
    away = _away(_device(target, tokens, u, u_next, draft, parents, tree_len, workspace, *(out or ())))
    if away is not None:
        with away:
            return verify_drafts(target, tokens, u, u_next, draft, parents, tree_len, out, workspace)
    if target.dim() != 3:
        raise ValueError("target must be [B, T, V]")
    B, T, V = target.shape
    if target.numel() > MOST:
        _sizes(B, T, V)
    code = _code(target)
    if target.stride(2) != 1 and V > 1:
        target = target.contiguous()
    if draft is not None:
        if draft.shape != target.shape or draft.dtype != target.dtype:
            raise ValueError(f"draft must be {target.dtype} {[B, T, V]}, got {draft.dtype} {list(draft.shape)}")
        if parents is not None:
            raise ValueError("draft probabilities are those of a chain: no parents")
        if draft.stride(2) != 1 and V > 1:
            draft = draft.contiguous()
    tokens = _packed(_ints("tokens", tokens, (B, T)))
    u, u_next = _floats("u", u, (B, T)), _floats("u_next", u_next, (B,))
    if parents is not None:
        parents = _packed(_ints("parents", parents, (B, T)))
    if tree_len is not None:
        tree_len = _packed(_ints("tree_len", tree_len, (B,)))
    if out is None:
        dev = target.device
        path, kept = torch.empty((B, T), dtype=torch.int32, device=dev), torch.empty(B, dtype=torch.int32, device=dev)
        token = torch.empty_like(kept)
    else:
        path, kept, token = out
        for name, t, shape in (("path", path, (B, T)), ("kept", kept, (B,)), ("token", token, (B,))):
            if not _ints(name, t, shape).is_contiguous():
                raise ValueError(f"{name} must be contiguous")
    workspace, at, size = _space(workspace, _verify_workspace(B, V), target.device)
    st = _lib.lib().ythip_verify_drafts(
        code, B, T, V, target.data_ptr(), _i64(target.stride()), None if draft is None else draft.data_ptr(),
        None if draft is None else _i64(draft.stride()), tokens.data_ptr(), T, None if parents is None else parents.data_ptr(),
        T, None if tree_len is None else tree_len.data_ptr(), u.data_ptr(), T, u_next.data_ptr(), path.data_ptr(), T,
        kept.data_ptr(), token.data_ptr(), at, size, _stream())
    if st:
        check(st, "ythip_verify_drafts")
    return path, kept, token
