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
makes the workspace).  A graph goes on using the workspace that it was captured
with, the eager call's: replay it in order with the calls of that stream.

What the device finds wrong (a length, page, parent or offset out of range) raises
on a later call on the stream, and on every one after it until :func:`status` has
read it.  A call that reads pages also raises what page calls on the stream have
reported (:func:`adakv_b200.paged.status`): after a refused append, say, it would
read lengths that are not what its caller takes them for.
"""
from __future__ import annotations

import math

import torch

from . import _lib


def _token_view(name, t, shape):
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)} (got {tuple(t.shape)})")
    st, sh, sd = t.stride()
    if sd != 1:
        raise ValueError(f"{name}: the head_dim axis must be contiguous")
    return _lib.pack_token_view(t.data_ptr(), st, sh)


def int32_vector(name, t, n, device):
    """Check a contiguous int32 vector of `n` entries on `device`; its address."""
    if t.dtype != torch.int32 or t.shape != (n,) or t.device != device:
        raise ValueError(f"{name} must be an int32 vector of {n} entries on {device} "
                         f"(got {t.dtype} {tuple(t.shape)} on {t.device})")
    if n > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def page_rows(page_table, seq_lens, device):
    """Check a page table ``[n_slots, width]`` with its lengths ``[n_slots]``:
    its address, row stride, width and rows, and the lengths' address."""
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.device != device:
        raise ValueError(f"page_table must be int32 [slots, width] on {device} "
                         f"(got {page_table.dtype} {tuple(page_table.shape)} on {page_table.device})")
    (rows, width), (stride, step) = page_table.shape, page_table.stride()
    if width > 1 and step != 1:
        raise ValueError("page_table rows must be contiguous")
    return (page_table.data_ptr(), stride, width, rows,
            int32_vector("seq_lens", seq_lens, rows, device))


def _prefix(k_pages, v_pages, page_table, seq_lens, slots, k, n_seqs):
    (_, Hkv, D), dtype, device = k.shape, k.dtype, k.device
    strides = []
    for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
        shape = t.shape
        if len(shape) != 4 or shape[1] != Hkv or shape[3] != D:
            raise ValueError(f"{name} must be [n_pages, {Hkv}, page_size, {D}] (got {tuple(shape)})")
        if t.dtype != dtype or t.device != device:
            raise ValueError(f"{name} must be {dtype} on {device}")
        sp, sh, st, sd = t.stride()
        if sd != 1:
            raise ValueError(f"{name}: the head_dim axis must be contiguous")
        strides += sp, sh, st
    if k_pages.shape != shape:
        raise ValueError("k_pages and v_pages must have one shape")
    table, stride, width, rows, lens = page_rows(page_table, seq_lens, device)
    at = int32_vector("slots", slots, n_seqs, device) if slots is not None else 0
    return _lib.pack_prefix(k_pages.data_ptr(), v_pages.data_ptr(), *strides, table, stride, lens,
                            at, width, rows, shape[0], shape[2])


def status(device) -> int:
    """Synchronise, return and clear the ``ST_*`` bits that attention calls on
    this stream of ``device`` have reported (0: none).  Until then each further
    one raises."""
    return _lib.stream_status(device, "extend")


_ws_bytes: dict = {}  # (device, dtype code, head_dim) -> bytes of workspace


def _attend(q, k, v, parents, cu_seqlens, pages, slots, scale, out, return_lse):
    if not q.is_cuda:
        _lib.require_cuda(q)
    dtype, device = q.dtype, q.device
    code = _lib.dtype_code(q)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k must be [tokens, heads, head_dim] (got {tuple(q.shape)}, "
                         f"{tuple(k.shape)})")
    shape = q.shape
    T, Hq, D = shape
    Hkv = k.shape[1]
    if k.dtype != dtype or v.dtype != dtype or k.device != device or v.device != device or \
            (out is not None and (out.dtype != dtype or out.device != device)):
        for name, t in (("k", k), ("v", v), ("out", out)):
            if t is not None and (t.dtype != dtype or t.device != device):
                raise ValueError(f"{name} must be {dtype} on {device} (got {t.dtype} on {t.device})")
    kv_shape = (T, Hkv, D)
    qv = _token_view("q", q, shape)
    kv = _token_view("k", k, kv_shape)
    vv = _token_view("v", v, kv_shape)
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be a vector of sequences + 1 offsets")
    n_seqs = cu_seqlens.shape[0] - 1
    cu = int32_vector("cu_seqlens", cu_seqlens, n_seqs + 1, device)
    par = int32_vector("parents", parents, T, device) if parents is not None else None
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        ov = _lib.pack_token_view(out.data_ptr(), Hq * D, D)
    else:
        ov = _token_view("out", out, shape)
    lse = q.new_empty((T, Hq), dtype=torch.float32) if return_lse else None
    prefix = None
    if pages is not None:
        prefix = _prefix(*pages, slots, k, n_seqs)
        _lib.raise_pending(device, "pages")
    if slots is not None and pages is None:
        raise ValueError("slots name rows of a page table: give the pages too")
    if T > 0 and n_seqs > 0:
        L = _lib.lib()
        key = (device.index, code, D)
        nbytes = _ws_bytes.get(key)
        if nbytes is None:
            with torch.cuda.device(device):
                nbytes = L.adakv_extend_workspace_bytes(code, D)
            if nbytes == 0:
                _lib.check(_lib.ERR_UNSUPPORTED)
            _ws_bytes[key] = nbytes
        _lib.run(L.adakv_extend_attend, device, "extend", nbytes,
                 _lib.pack_new_tokens(n_seqs, T, Hq, Hkv, D, code), qv, kv, vv, cu, par, prefix,
                 scale, ov, lse.data_ptr() if return_lse else None)
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
    lse -inf, and nothing attends to it).  At most 65536 drafted tokens, and meant
    for trees of some hundred: a row walks its ancestors for every 64 drafted
    tokens before it (a long chain is a prompt).  The other arguments are those of
    :func:`prompt_attention`."""
    if parents is None:
        raise ValueError("parents are needed (prompt_attention is the causal form)")
    return _attend(q, k, v, parents, cu_seqlens, (k_pages, v_pages, page_table, seq_lens), slots,
                   scale, out, return_lse)
