"""Calls of the paged cache: empty lists, lists of the host, and who learns of a
request that could not be met."""
import pytest
import torch

from adakv_b200 import _lib, paged
from adakv_b200.paged import PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    paged.status("cuda:0")  # bits of an earlier test


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cache(n_pages=8, n_slots=4, max_seq_len=64, **kw):
    return PagedKVCache(2, n_pages, 2, 64, 16, n_slots, max_seq_len, torch.bfloat16, "cuda", **kw)


def new(n, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((2, n, 2, 64), generator=g).to(torch.bfloat16).cuda()


def test_index_of_no_width_accepts_nothing():
    """``index`` [B, 0]: no drafted token was accepted, nothing is written."""
    c = cache()
    k = new(6)
    c.append(k, k, i32([0, 6]), slots=i32([1]))
    before = c.page_table.clone()
    c.append(k, k, i32([0, 2, 6]), slots=i32([0, 1]), index=torch.empty((2, 0), dtype=torch.int32, device="cuda"),
             counts=i32([0, 0]))
    c.append(k, k, i32([0, 2, 6]), slots=i32([0, 1]), index=torch.empty((2, 0), dtype=torch.int32, device="cuda"))
    assert c.status() == 0
    assert c.seq_lens.tolist() == [0, 6, 0, 0] and torch.equal(c.page_table, before)
    # a count that the index does not hold is still an error
    c.append(k, k, i32([0, 2, 6]), slots=i32([0, 1]), index=torch.empty((2, 0), dtype=torch.int32, device="cuda"),
             counts=i32([0, 1]))
    assert c.status() == _lib.ST_BAD_SEQ_LEN
    assert c.seq_lens.tolist() == [0, 6, 0, 0]


def test_lists_of_the_host_do_not_synchronise():
    """fork, free and copy with lists, as a server calls them: no wait for the GPU."""
    c = cache(n_pages=20, n_slots=12)
    k = new(40)
    c.append(k, k, i32([0, 40]), slots=i32([1]))
    c.fork([1], [2])  # (page-locked memory is allocated once)
    torch.cuda.synchronize()
    try:
        torch.cuda.set_sync_debug_mode("error")
        c.fork([1, 2], [3, 5])
        c.free([2, 2])
        c.free([])
        c.copy([0, 1], [10, 11])
        c.free(range(5, 6))
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert c.status() == 0
    assert c.seq_lens.tolist() == [0, 40, 0, 40] + [0] * 8
    assert torch.equal(c.k[:, 10:12], c.k[:, 0:2]) and torch.equal(c.v[:, 10:12], c.v[:, 0:2])


def test_many_lists_in_flight():
    """Lists given one after the other while the GPU is behind: each call has its own."""
    c = cache(n_pages=64, n_slots=64)
    c.refcounts.fill_(1)
    c.page_table[:, 0] = torch.arange(64, dtype=torch.int32, device="cuda")
    c.seq_lens.fill_(16)
    busy = torch.randn(4096, 4096, device="cuda")
    for _ in range(20):
        busy = busy @ busy * 1e-3
    for s in range(0, 64, 2):
        c.free([s])
    assert c.status() == 0
    assert c.seq_lens.tolist() == [0, 16] * 32 and c.refcounts.tolist() == [0, 1] * 32


def test_lists_are_refused_while_a_graph_is_captured():
    c = cache()
    k = new(20)
    c.append(k, k, i32([0, 20]), slots=i32([1]))
    src, dst = i32([1]), i32([2])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: c.fork([1], [2]), lambda: c.free([1]), lambda: c.copy([0], [1])):
            with pytest.raises(ValueError, match="captured"):
                call()
        c.fork(src, dst)
    graph.replay()
    assert c.status() == 0 and c.seq_lens.tolist() == [0, 20, 20, 0]
    del graph
