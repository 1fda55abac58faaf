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
