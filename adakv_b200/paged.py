"""A paged KV cache: pages that sequences share, fork, give back and fill.

``k`` / ``v`` are pools ``[n_layers, n_pages, n_kv_heads, page_size, head_dim]``.
Row s of ``page_table`` (int32 ``[n_slots, width]``, -1 behind the last page)
names sequence s's pages in order, ``seq_lens[s]`` its tokens, ``refcounts[p]``
how many rows name page p (0: free).  All of it lies on the GPU and is changed
there: no call synchronises, and all can be captured in a CUDA graph (the
functions after one eager call, which makes the stream's workspace; a graph goes on
using that one: replay it in order with the calls of that stream).

Full pages are shared between forks; the last, partly filled page of a sequence
is always its own.  Free pages are taken lowest id first in the order of the
request, so results do not depend on timing.  A fork or append that names a bad
row, or that needs more pages than are free, changes nothing; once the GPU has
found that out, the next call on the stream raises, and so does attention that
reads pages, until :func:`status` has read the bits (it waits for them).

The functions work on plain tensors, :class:`PagedKVCache` owns a set of them.
"""
from __future__ import annotations

import torch

from . import _lib
from .prompt import int32_vector, page_rows, prompt_attention
from .prompt import status as attention_status
from .prompt import tree_attention


def _run(own, fn, device, n_pages, *args):
    """``fn`` with a cache's own workspace, or (None) with the stream's."""
    if own is not None:
        own.run(fn, *args)
    else:
        _lib.run(fn, device, "pages", _bytes(n_pages), *args)


def _pool(k, v):
    if not k.is_cuda or not v.is_cuda:
        _lib.require_cuda(k, v)
    shape, k_strides, v_strides = k.shape, k.stride(), v.stride()
    if len(shape) != 5 or v.dim() != 5:
        raise ValueError("k and v must be [layers, pages, heads, page_size, head_dim] "
                         f"(got {tuple(shape)}, {tuple(v.shape)})")
    _, _, H, ps, D = shape
    if v.shape != shape or k.dtype != v.dtype or k.device != v.device:
        raise ValueError("k and v must have one shape, type and device")
    for name, (_, _, sh, ss, sd) in (("k", k_strides), ("v", v_strides)):
        if sd != 1 or (ss != D and ps > 1) or (sh != ps * D and H > 1):
            raise ValueError(f"{name}: a page [heads, page_size, head_dim] must be contiguous")
    return _lib.pack_page_pool(k.data_ptr(), v.data_ptr(), k_strides[0], k_strides[1], v_strides[0],
                               v_strides[1], *shape, _lib.dtype_code(k))


def _table(page_table, seq_lens, refcounts, n_pages, device):
    if not page_table.is_cuda:
        _lib.require_cuda(page_table)
    table, stride, width, rows, lens = page_rows(page_table, seq_lens, device)
    return _lib.pack_page_table(table, stride, lens,
                                int32_vector("refcounts", refcounts, n_pages, device), width, rows)


def _lists(a, b, device, names):
    n = a.shape[0] if a.dim() == 1 else -1
    return int32_vector(names[0], a, n, device), int32_vector(names[1], b, n, device), n


_ws_bytes: dict = {}  # pages of a pool -> bytes of workspace


def _bytes(n_pages):
    nbytes = _ws_bytes.get(n_pages)
    if nbytes is None:
        nbytes = _lib.lib().adakv_pages_workspace_bytes(n_pages)
        if nbytes == 0:
            _lib.check(_lib.ERR_INVALID)
        _ws_bytes[n_pages] = nbytes
    return nbytes


def status(device) -> int:
    """Synchronise, return and clear the ``ST_*`` bits that page calls on this
    stream of ``device`` have reported (0: none)."""
    return _lib.stream_status(device, "pages")


def copy_pages(k, v, src, dst):
    """Page ``dst[i]`` becomes a copy of page ``src[i]``, in every layer, k and v.
    ``dst`` must name no page twice and none of ``src``."""
    _copy(None, k, v, src, dst)


def _copy(own, k, v, src, dst):
    pool, device = _pool(k, v), k.device
    _run(own, _lib.lib().adakv_pages_copy, device, k.shape[1], pool,
         *_lists(src, dst, device, ("src", "dst")))


def fork_sequences(k, v, page_table, seq_lens, refcounts, src, dst):
    """Row ``dst[i]``, which must be empty, becomes a copy of row ``src[i]``: the
    full pages are shared, the partly filled last one is copied to a free page."""
    _fork(None, k, v, page_table, seq_lens, refcounts, src, dst)


def _fork(own, k, v, page_table, seq_lens, refcounts, src, dst):
    pool, device, n_pages = _pool(k, v), k.device, k.shape[1]
    table = _table(page_table, seq_lens, refcounts, n_pages, device)
    _run(own, _lib.lib().adakv_pages_fork, device, n_pages, pool, table,
         *_lists(src, dst, device, ("src", "dst")))


def free_sequences(page_table, seq_lens, refcounts, slots):
    """The rows ``slots`` give their pages back and are empty afterwards."""
    _free(None, page_table, seq_lens, refcounts, slots)


def _free(own, page_table, seq_lens, refcounts, slots):
    n_pages, device = refcounts.shape[0], page_table.device
    table = _table(page_table, seq_lens, refcounts, n_pages, device)
    n = slots.shape[0] if slots.dim() == 1 else -1
    _run(own, _lib.lib().adakv_pages_free, device, n_pages, table, n_pages,
         int32_vector("slots", slots, n, device), n)


def compact_pages(k, v, page_table, seq_lens, refcounts):
    """Make the pool dense: with L live pages, the i-th live page with an id of L
    or more moves to the i-th free one below L."""
    _compact(None, k, v, page_table, seq_lens, refcounts)


def _compact(own, k, v, page_table, seq_lens, refcounts):
    pool, device, n_pages = _pool(k, v), k.device, k.shape[1]
    table = _table(page_table, seq_lens, refcounts, n_pages, device)
    _run(own, _lib.lib().adakv_pages_compact, device, n_pages, pool, table)


def append_tokens(k, v, page_table, seq_lens, refcounts, k_new, v_new, cu_seqlens, *, slots=None,
                  index=None, counts=None):
    """Write new tokens behind those that the sequences hold, on fresh pages
    where theirs are full.

    ``k_new`` / ``v_new`` ``[layers, T, heads, head_dim]``; sequence b's tokens
    are ``[cu_seqlens[b], cu_seqlens[b + 1])`` of them.  Written are all of them,
    or the first ``counts[b]``, or (``index`` int32 ``[B, W]``) those at the
    positions ``index[b, :counts[b]]`` among them, in that order: the accepted
    path of a drafted tree (a width of 0: nothing)."""
    _append(None, k, v, page_table, seq_lens, refcounts, k_new, v_new, cu_seqlens, slots, index, counts)


def _append(own, k, v, page_table, seq_lens, refcounts, k_new, v_new, cu_seqlens, slots, index, counts):
    pool, device = _pool(k, v), k.device
    L, n_pages, H, _, D = k.shape
    table = _table(page_table, seq_lens, refcounts, n_pages, device)
    views = []
    for name, t in (("k_new", k_new), ("v_new", v_new)):
        if t.dim() != 4 or (t.shape[0], t.shape[2], t.shape[3]) != (L, H, D):
            raise ValueError(f"{name} must be [{L}, tokens, {H}, {D}] (got {tuple(t.shape)})")
        if t.dtype != k.dtype or t.device != device:
            raise ValueError(f"{name} must be {k.dtype} on {device}")
        sl, st, sh, sd = t.stride()
        if sd != 1:
            raise ValueError(f"{name}: the head_dim axis must be contiguous")
        views.append(_lib.pack_layer_tokens(t.data_ptr(), sl, st, sh))
    if k_new.shape != v_new.shape:
        raise ValueError("k_new and v_new must have one shape")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("cu_seqlens must be a vector of sequences + 1 offsets")
    B = cu_seqlens.shape[0] - 1
    cu = int32_vector("cu_seqlens", cu_seqlens, B + 1, device)
    rows = int32_vector("slots", slots, B, device) if slots is not None else None
    cnt = int32_vector("counts", counts, B, device) if counts is not None else None
    idx, idx_stride, width = None, 0, 0
    if index is not None:
        if index.dtype != torch.int32 or index.dim() != 2 or index.shape[0] != B or \
                index.device != device or (index.shape[1] > 1 and index.stride(1) != 1):
            raise ValueError(f"index must be int32 [{B}, width] with contiguous rows on {device} "
                             f"(got {index.dtype} {tuple(index.shape)} on {index.device})")
        # (an index of no width has no address, but is not the same as none)
        idx, idx_stride, width = index.data_ptr() or cu, index.stride(0), index.shape[1]
    if B > 0 and k_new.shape[1] > 0:
        _run(own, _lib.lib().adakv_pages_append, device, n_pages, pool, table, B,
             k_new.shape[1], *views, cu, rows, idx, idx_stride, width, cnt)


class PagedKVCache:
    """Pools for ``n_layers`` layers, with the page table, lengths and reference
    counts of up to ``n_slots`` sequences of ``max_seq_len`` tokens.

    The status of its page calls is the cache's own: what one of them reports
    raises on the next call of this cache, attention included, and of no other.
    They change one set of tables, so those on several streams need to be ordered
    by their caller."""

    def __init__(self, n_layers, n_pages, n_kv_heads, head_dim, page_size=16, n_slots=64,
                 max_seq_len=32768, dtype=torch.bfloat16, device="cuda"):
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page_size must be 16, 32, 64 or 128 (got {page_size})")
        if head_dim not in (64, 128):
            raise NotImplementedError(f"head_dim must be 64 or 128 (got {head_dim})")
        if min(n_layers, n_pages, n_kv_heads, n_slots, max_seq_len) < 1:
            raise ValueError("layers, pages, heads, slots and max_seq_len must be 1 or more")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("adakv_b200 runs on CUDA tensors only (no CPU fallback)")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        _lib.dtype_code(self.k)
        self.page_size = page_size
        self.max_pages = -(-max_seq_len // page_size)
        self.page_table = torch.full((n_slots, self.max_pages), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(n_slots, dtype=torch.int32, device=device)
        self.refcounts = torch.zeros(n_pages, dtype=torch.int32, device=device)
        self._own = _lib.OwnWorkspace(_bytes(n_pages), device)

    @property
    def _owned(self):
        return self.page_table, self.seq_lens, self.refcounts

    def layer(self, i):
        """``(k_pages, v_pages, page_table, seq_lens)`` of layer i, as
        :func:`~adakv_b200.prompt.prompt_attention` and
        :func:`~adakv_b200.prompt.tree_attention` take it.  Raises what page calls
        on this cache have reported."""
        self._own.sink.raise_if_set()
        return self.k[i], self.v[i], self.page_table, self.seq_lens

    def _ids(self, x):
        """Rows or pages as an int32 tensor on the device; a list is copied there
        from page-locked memory, in stream order."""
        if isinstance(x, torch.Tensor):
            return x
        x = list(x)
        if not x:
            return torch.empty(0, dtype=torch.int32, device=self.k.device)
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("while a graph is captured, rows and pages have to be int32 tensors on the "
                             "device (a list's memory is not kept for the replays)")
        return torch.tensor(x, dtype=torch.int32, pin_memory=True).to(self.k.device, non_blocking=True)

    def prompt_attention(self, layer, q, k, v, cu_seqlens, **kw):
        """:func:`~adakv_b200.prompt.prompt_attention` after what is cached."""
        return prompt_attention(q, k, v, cu_seqlens, self.layer(layer), **kw)

    def tree_attention(self, layer, q, k, v, parents, cu_seqlens, **kw):
        """:func:`~adakv_b200.prompt.tree_attention` over what is cached."""
        return tree_attention(q, k, v, parents, cu_seqlens, *self.layer(layer), **kw)

    def append(self, k_new, v_new, cu_seqlens, *, slots=None, index=None, counts=None):
        """:func:`append_tokens`."""
        _append(self._own, self.k, self.v, *self._owned, k_new, v_new, cu_seqlens, slots, index, counts)

    def fork(self, src, dst):
        """:func:`fork_sequences`; rows as an int32 tensor on the device, or as a
        list (not while a graph is captured)."""
        _fork(self._own, self.k, self.v, *self._owned, self._ids(src), self._ids(dst))

    def free(self, slots):
        """:func:`free_sequences`; rows as :meth:`fork` takes them."""
        _free(self._own, *self._owned, self._ids(slots))

    def compact(self):
        """:func:`compact_pages`."""
        _compact(self._own, self.k, self.v, *self._owned)

    def copy(self, src, dst):
        """:func:`copy_pages`; pages as :meth:`fork` takes rows."""
        _copy(self._own, self.k, self.v, self._ids(src), self._ids(dst))

    def status(self) -> int:
        """Synchronise, return and clear the status bits of this cache's page calls
        and of attention on this stream."""
        return self._own.status() | attention_status(self.k.device)
