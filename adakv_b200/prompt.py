"""Attention of new tokens: whole prompts, and trees of drafted tokens.

* :func:`prompt_attention`: causal attention of packed prompts of different
  lengths, with grouped heads, each optionally after tokens that lie in a paged
  cache already (the next piece of a chunked prompt).
* :func:`tree_attention`: attention of each sequence's drafted tokens (a tree,
  given by parents) over its paged cache and their own ancestors; one drafted
  token per sequence is an ordinary decode step.

Both are one call of ``adakv_extend_attend``.  The new tokens' keys and values
are arguments of their own: nothing has to be in the cache before it is known
to stay (:func:`adakv_b200.paged.append_tokens` writes what is accepted).

Inference only: the outputs carry no gradient.  Work is enqueued on the current
stream; lengths, parents and pages are read on the device, so the calls never
synchronise and can be captured in a CUDA graph (after one eager call, which
makes the workspace).
"""
from __future__ import annotations

import math

import torch

from . import _lib


def _token_view(name, t, heads=None, dim=None, tokens=None):
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim] (got {tuple(t.shape)})")
    if tokens is not None and (t.shape[0], t.shape[1], t.shape[2]) != (tokens, heads, dim):
        raise ValueError(f"{name} must be [{tokens}, {heads}, {dim}] (got {tuple(t.shape)})")
    if t.stride(2) != 1:
        raise ValueError(f"{name}: the head_dim axis must be contiguous")
    return _lib.TokenView(t.data_ptr(), t.stride(0), t.stride(1))


def int32_vector(name, t, n, device):
    """Check a contiguous int32 vector of `n` entries on `device`; its address."""
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or t.device != device:
        raise ValueError(f"{name} must be an int32 vector of {n} entries on {device} "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def page_rows(page_table, seq_lens, device):
    """Check a page table ``[n_slots, width]`` with its lengths ``[n_slots]``."""
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.device != device:
        raise ValueError(f"page_table must be int32 [slots, width] on {device} "
                         f"(got {page_table.dtype} {tuple(page_table.shape)} on {page_table.device})")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("page_table rows must be contiguous")
    int32_vector("seq_lens", seq_lens, page_table.shape[0], device)


def _prefix(k_pages, v_pages, page_table, seq_lens, slots, k, n_seqs):
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        if t.dim() != 4 or t.shape[1] != k.shape[1] or t.shape[3] != k.shape[2]:
            raise ValueError(f"{name} must be [n_pages, {k.shape[1]}, page_size, {k.shape[2]}] "
                             f"(got {tuple(t.shape)})")
        if t.dtype != k.dtype or t.device != k.device:
            raise ValueError(f"{name} must be {k.dtype} on {k.device}")
        if t.stride(3) != 1:
            raise ValueError(f"{name}: the head_dim axis must be contiguous")
    if k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must have one shape")
    page_rows(page_table, seq_lens, k.device)
    return _lib.Prefix(k_pages.data_ptr(), v_pages.data_ptr(), k_pages.stride(0), k_pages.stride(1),
                       k_pages.stride(2), v_pages.stride(0), v_pages.stride(1), v_pages.stride(2),
                       page_table.data_ptr(), page_table.stride(0), seq_lens.data_ptr(),
                       int32_vector("slots", slots, n_seqs, k.device) if slots is not None else None,
                       page_table.shape[1], page_table.shape[0], k_pages.shape[0], k_pages.shape[2])


def _attend(q, k, v, parents, cu_seqlens, pages, slots, scale, out, return_lse):
    _lib.require_cuda(q, k, v, parents, cu_seqlens, out)
    code = _lib.dtype_code(q)
    qv = _token_view("q", q)
    T, Hq, D = q.shape
    kv = _token_view("k", k, k.shape[1] if k.dim() == 3 else 0, D, T)
    Hkv = k.shape[1]
    vv = _token_view("v", v, Hkv, D, T)
    device = q.device
    for name, t in (("k", k), ("v", v), ("out", out)):
        if t is not None and (t.dtype != q.dtype or t.device != device):
            raise ValueError(f"{name} must be {q.dtype} on {device} (got {t.dtype} on {t.device})")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be a vector of sequences + 1 offsets")
    n_seqs = cu_seqlens.shape[0] - 1
    cu = int32_vector("cu_seqlens", cu_seqlens, n_seqs + 1, device)
    par = int32_vector("parents", parents, T, device) if parents is not None else None
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((T, Hq, D), dtype=q.dtype, device=device)
    ov = _token_view("out", out, Hq, D, T)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=device) if return_lse else None
    prefix = _prefix(*pages, slots, k, n_seqs) if pages is not None else None
    if slots is not None and pages is None:
        raise ValueError("slots name rows of a page table: give the pages too")
    if T > 0 and n_seqs > 0:
        L = _lib.lib()
        geo = _lib.NewTokens(n_seqs, T, Hq, Hkv, D, code)
        with torch.cuda.device(device):
            nbytes = L.adakv_extend_workspace_bytes(geo)
            if nbytes == 0:
                # the call itself names what is wrong with the geometry
                _lib.check(L.adakv_extend_attend(geo, qv, kv, vv, cu, par, prefix, scale, ov, None,
                                                 None, 0, None))
            ws = _lib.workspace(nbytes, device, "extend")
            _lib.raise_if_failed(ws)
            _lib.check(L.adakv_extend_attend(geo, qv, kv, vv, cu, par, prefix, scale, ov,
                                             lse.data_ptr() if return_lse else None, ws.data_ptr(),
                                             ws.numel(), _lib.stream_ptr(device)))
    return (out, lse) if return_lse else out


def prompt_attention(q, k, v, cu_seqlens, prefix=None, *, slots=None, scale=None, out=None,
                     return_lse=False):
    """Causal attention of packed prompts.

    ``q`` ``[T, Hq, D]``, ``k`` / ``v`` ``[T, Hkv, D]`` (any token and head
    strides of whole 16-byte words), ``cu_seqlens`` int32 ``[B + 1]``: sequence
    b's tokens are ``[cu_seqlens[b], cu_seqlens[b + 1])``, none included.
    ``prefix`` is ``(k_pages, v_pages, page_table, seq_lens)`` (of one layer:
    :meth:`adakv_b200.paged.PagedKVCache.layer`): tokens of the same sequences
    that every new one attends to as well; ``slots`` int32 ``[B]`` names the
    sequences' rows of the page table (default: sequence b has row b).

    Returns ``out`` ``[T, Hq, D]``, with ``return_lse`` also the float32 ``[T,
    Hq]`` natural log of each row's sum of exp.  Rows of ``q`` outside every
    sequence are not written."""
    return _attend(q, k, v, None, cu_seqlens, prefix, slots, scale, out, return_lse)


def tree_attention(q, k, v, parents, cu_seqlens, k_pages, v_pages, page_table, seq_lens, *,
                   slots=None, scale=None, out=None, return_lse=False):
    """Attention of drafted tokens over a paged cache and their own ancestors.

    ``parents`` int32 ``[T]``: the position of each drafted token's parent
    among its sequence's drafted tokens, which must lie before it; -1: it
    follows the last cached token; -2: the slot is unused (its ``out`` is 0, its
    lse -inf, and nothing attends to it).  The other arguments are those of
    :func:`prompt_attention`."""
    if parents is None:
        raise ValueError("parents are needed (prompt_attention is the causal form)")
    return _attend(q, k, v, parents, cu_seqlens, (k_pages, v_pages, page_table, seq_lens), slots,
                   scale, out, return_lse)
