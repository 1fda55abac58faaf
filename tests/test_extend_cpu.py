"""Refusals of the new-token attention and page entry points that need no GPU:
arguments are checked before anything is launched."""
from __future__ import annotations

import pytest
import torch

from adakv_b200 import _lib, paged, prompt
from adakv_b200.build import build


@pytest.fixture(scope="module")
def lib():
    build()
    return _lib.lib()


P = 0x10000  # a 16-byte aligned address that is never read


def tokens(**kw):
    d = dict(n_seqs=1, n_tokens=4, n_q_heads=8, n_kv_heads=2, head_dim=64, dtype=_lib.DTYPE_BF16)
    d.update(kw)
    return _lib.pack_new_tokens(*d.values())


def prefix(**kw):
    d = dict(k=P, v=P, ksp=4096, ksh=1024, kst=64, vsp=4096, vsh=1024, vst=64, table=P, stride=8,
             lens=P, slots=0, width=8, n_slots=3, n_pages=9, page_size=16)
    d.update(kw)
    return _lib.pack_prefix(*d.values())


VIEW = _lib.pack_token_view(P, 512, 64)


def attend(lib, geo=None, q=VIEW, k=VIEW, v=VIEW, cu=P, parents=None, pre=None, scale=0.125, out=VIEW):
    return lib.adakv_extend_attend(geo or tokens(), q, k, v, cu, parents, pre, scale, out, None, P, 0, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(geo=tokens(n_seqs=0)), _lib.ERR_INVALID, "n_seqs"),
    (dict(geo=tokens(n_tokens=0)), _lib.ERR_INVALID, "n_tokens"),
    (dict(geo=tokens(n_q_heads=7)), _lib.ERR_INVALID, "multiple"),
    (dict(geo=tokens(n_q_heads=256)), _lib.ERR_UNSUPPORTED, "group"),
    (dict(geo=tokens(head_dim=96)), _lib.ERR_UNSUPPORTED, "head_dim"),
    (dict(geo=tokens(dtype=7)), _lib.ERR_INVALID, "dtype"),
    (dict(q=None), _lib.ERR_INVALID, "q is NULL"),
    (dict(k=_lib.pack_token_view(0, 512, 64)), _lib.ERR_INVALID, "k is NULL"),
    (dict(v=_lib.pack_token_view(P + 2, 512, 64)), _lib.ERR_INVALID, "aligned"),
    (dict(q=_lib.pack_token_view(P, 516, 64)), _lib.ERR_INVALID, "16 bytes"),
    (dict(k=_lib.pack_token_view(P, 0, 64)), _lib.ERR_INVALID, "positive"),
    (dict(out=_lib.pack_token_view(P, -512, 64)), _lib.ERR_INVALID, "positive"),
    (dict(cu=None), _lib.ERR_INVALID, "cu_new"),
    (dict(geo=tokens(n_tokens=1 << 29)), _lib.ERR_UNSUPPORTED, "group size"),
    (dict(geo=tokens(n_tokens=65537), parents=P), _lib.ERR_UNSUPPORTED, "drafted"),
    (dict(scale=0.0), _lib.ERR_INVALID, "scale"),
    (dict(scale=float("nan")), _lib.ERR_INVALID, "scale"),
    (dict(pre=prefix(page_size=8)), _lib.ERR_UNSUPPORTED, "page_size"),
    (dict(pre=prefix(n_pages=0)), _lib.ERR_INVALID, "pages"),
    (dict(pre=prefix(table=0)), _lib.ERR_INVALID, "page_table"),
    (dict(pre=prefix(lens=0)), _lib.ERR_INVALID, "seq_lens"),
    (dict(pre=prefix(stride=7)), _lib.ERR_INVALID, "overlap"),
    (dict(pre=prefix(kst=60)), _lib.ERR_INVALID, "16 bytes"),
    (dict(pre=prefix(vsp=0)), _lib.ERR_INVALID, "positive"),
    (dict(pre=prefix(width=1 << 28)), _lib.ERR_UNSUPPORTED, "2\\^30"),
    (dict(geo=tokens(n_seqs=4), pre=prefix()), _lib.ERR_INVALID, "slots"),
])
def test_attend_refusals(lib, kw, code, text):
    assert attend(lib, **kw) == code
    assert pytest.importorskip("re").search(text, lib.adakv_last_error().decode())


def pool(**kw):
    d = dict(k=P, v=P, ksl=1 << 20, ksp=4096, vsl=1 << 20, vsp=4096, layers=2, pages=64, heads=4,
             page_size=16, head_dim=64, dtype=_lib.DTYPE_BF16)
    d.update(kw)
    return _lib.pack_page_pool(*d.values())


def table(**kw):
    d = dict(table=P, stride=8, lens=P, ref=P, width=8, n_slots=3)
    d.update(kw)
    return _lib.pack_page_table(*d.values())


WS = 256 + (1 << 20)


@pytest.mark.parametrize("kw,code,text", [
    (dict(layers=0), _lib.ERR_INVALID, "layers"),
    (dict(pages=(1 << 20) + 1), _lib.ERR_UNSUPPORTED, "n_pages"),
    (dict(page_size=24), _lib.ERR_UNSUPPORTED, "page_size"),
    (dict(head_dim=80), _lib.ERR_UNSUPPORTED, "head_dim"),
    (dict(dtype=-1), _lib.ERR_INVALID, "dtype"),
    (dict(k=0), _lib.ERR_INVALID, "pool k"),
    (dict(v=P + 8), _lib.ERR_INVALID, "aligned"),
    (dict(ksp=4095), _lib.ERR_INVALID, "16 bytes"),
    (dict(vsp=2048), _lib.ERR_INVALID, "overlap"),
])
def test_pool_refusals(lib, kw, code, text):
    for call in (lambda x: lib.adakv_pages_copy(x, P, P, 1, P, WS, None),
                 lambda x: lib.adakv_pages_fork(x, table(), P, P, 1, P, WS, None),
                 lambda x: lib.adakv_pages_compact(x, table(), P, WS, None)):
        assert call(pool(**kw)) == code
        assert text in lib.adakv_last_error().decode()


def test_table_and_list_refusals(lib):
    bad = lib.adakv_last_error
    assert lib.adakv_pages_free(table(width=0), 64, P, 1, P, WS, None) == _lib.ERR_INVALID
    assert lib.adakv_pages_free(table(ref=0), 64, P, 1, P, WS, None) == _lib.ERR_INVALID
    assert lib.adakv_pages_free(table(stride=4), 64, P, 1, P, WS, None) == _lib.ERR_INVALID
    assert "overlap" in bad().decode()
    assert lib.adakv_pages_free(table(n_slots=1 << 17), 64, P, 1, P, WS, None) == _lib.ERR_UNSUPPORTED
    assert lib.adakv_pages_free(table(), 0, P, 1, P, WS, None) == _lib.ERR_INVALID
    assert lib.adakv_pages_free(table(), 64, None, 1, P, WS, None) == _lib.ERR_INVALID
    assert lib.adakv_pages_free(table(), 64, P, -1, P, WS, None) == _lib.ERR_INVALID
    assert lib.adakv_pages_copy(pool(), P, P, 1, P, 256, None) == _lib.ERR_INVALID
    assert "too small" in bad().decode()
    assert lib.adakv_pages_copy(pool(), P, P, 1, P + 16, WS, None) == _lib.ERR_INVALID
    assert lib.adakv_pages_fork(pool(), table(), P, P, 5000, P, WS, None) == _lib.ERR_UNSUPPORTED
    # nothing to do is no error
    assert lib.adakv_pages_copy(pool(), None, None, 0, P, WS, None) == _lib.OK
    assert lib.adakv_pages_free(table(), 64, None, 0, P, WS, None) == _lib.OK
    row = _lib.pack_layer_tokens(P, 4096, 256, 64)

    def append(n_seqs=2, n_tokens=8, k=row, v=row, cu=P, slots=None, index=None, stride=0, width=0):
        return lib.adakv_pages_append(pool(), table(), n_seqs, n_tokens, k, v, cu, slots, index,
                                      stride, width, None, P, WS, None)

    assert append(n_seqs=4) == _lib.ERR_INVALID and "slots" in bad().decode()
    assert append(cu=None) == _lib.ERR_INVALID
    assert append(k=None) == _lib.ERR_INVALID
    assert append(index=P, stride=2, width=3) == _lib.ERR_INVALID and "index" in bad().decode()
    assert append(v=_lib.pack_layer_tokens(P, 4096, 252, 64)) == _lib.ERR_INVALID
    assert append(n_tokens=-1) == _lib.ERR_INVALID
    assert append(n_tokens=0) == _lib.OK


def test_workspace_sizes(lib):
    assert lib.adakv_pages_workspace_bytes(0) == 0
    assert lib.adakv_pages_workspace_bytes((1 << 20) + 1) == 0
    a, b = (lib.adakv_pages_workspace_bytes(n) for n in (1, 1 << 20))
    assert 0 < a < b and a % 256 == 0 and b % 256 == 0
    assert lib.adakv_extend_workspace_bytes(_lib.DTYPE_BF16, 80) == 0


def test_no_cpu_fallback():
    q = torch.zeros(4, 8, 64)
    k = torch.zeros(4, 2, 64)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt.prompt_attention(q, k, k, cu)
    pages = torch.zeros(1, 4, 2, 16, 64)
    ids = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.copy_pages(pages, pages, ids, ids)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.free_sequences(ids[None], ids, ids, ids)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.PagedKVCache(1, 4, 1, 64, device="cpu")
