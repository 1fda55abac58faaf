"""Who learns of what the device found wrong, and how it is put right, through the
public calls alone."""
import pytest
import torch

from adakv_b200 import _lib, paged, prompt
from adakv_b200.prompt import prompt_attention, tree_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rnd(*shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def test_attention_recovers_from_a_bad_parent():
    q, k = rnd(3, 4, 64, seed=1), rnd(3, 2, 64, seed=2)
    kp = rnd(4, 2, 16, 64, seed=3)
    pages = (kp, kp, i32([[0, 1, 2]]), i32([40]))
    cu = i32([0, 3])
    prompt.status("cuda:0")
    want = tree_attention(q, k, k, i32([-1, 0, 1]), cu, *pages)
    tree_attention(q, k, k, i32([-1, 2, 1]), cu, *pages)
    torch.cuda.synchronize()
    for _ in range(2):
        with pytest.raises(RuntimeError, match="parent"):
            tree_attention(q, k, k, i32([-1, 0, 1]), cu, *pages)
        with pytest.raises(RuntimeError, match="parent"):
            prompt_attention(q, k, k, cu)
    assert prompt.status("cuda") == _lib.ST_BAD_PARENT
    assert prompt.status("cuda:0") == 0
    assert torch.equal(tree_attention(q, k, k, i32([-1, 0, 1]), cu, *pages), want)


def test_status_is_the_streams():
    q, k = rnd(3, 4, 64, seed=1), rnd(3, 2, 64, seed=2)
    prompt.status("cuda:0")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        prompt.status("cuda:0")
        prompt_attention(q, k, k, i32([0, 9]))
        s.synchronize()
    prompt_attention(q, k, k, i32([0, 3]))  # another stream's failure is not this one's
    assert prompt.status("cuda:0") == 0
    with torch.cuda.stream(s):
        assert prompt.status(torch.device("cuda")) == _lib.ST_BAD_SEQ_LEN


@pytest.mark.parametrize("device", ["cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0)], ids=str)
def test_page_status_by_any_name_of_the_device(device):
    paged.status("cuda:0")
    k = torch.zeros((1, 4, 1, 16, 64), dtype=torch.bfloat16, device="cuda")
    paged.copy_pages(k, k.clone(), i32([9]), i32([1]))
    assert paged.status(device) == _lib.ST_BAD_BLOCK_ID
    assert paged.status(device) == 0
    paged.copy_pages(k, k.clone(), i32([0]), i32([1]))


@pytest.mark.parametrize("tree", [True, False])
def test_attention_raises_a_refused_append(tree):
    """After an append that found no free pages, attention over the pages would run on
    the old lengths: it raises, like the next page call."""
    paged.status("cuda:0")
    k, v = (torch.zeros((1, 3, 2, 16, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    meta = [torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"),
            torch.zeros(3, dtype=torch.int32, device="cuda")]
    kn = rnd(1, 40, 2, 64, seed=1)
    paged.append_tokens(k, v, *meta, kn, kn, i32([0, 40]))
    paged.append_tokens(k, v, *meta, kn, kn, i32([0, 40]))  # 80 tokens need five pages
    torch.cuda.synchronize()
    q, cu = rnd(3, 4, 64, seed=2), i32([0, 3])

    def attend():
        if tree:
            return tree_attention(q, kn[0, :3], kn[0, :3], i32([-1, 0, 1]), cu, k[0], v[0], meta[0], meta[1])
        return prompt_attention(q, kn[0, :3], kn[0, :3], cu, (k[0], v[0], meta[0], meta[1]))

    with pytest.raises(RuntimeError, match="free pages"):
        attend()
    prompt_attention(q, kn[0, :3], kn[0, :3], cu)  # no pages are read
    assert paged.status("cuda:0") == _lib.ST_NO_PAGES
    attend()
    assert prompt.status("cuda:0") == 0


def caches(n):
    return [paged.PagedKVCache(1, 3, 2, 64, 16, 2, 128, torch.bfloat16, "cuda") for _ in range(n)]


def test_a_caches_failure_is_its_own():
    """A refused append on one cache: that cache's next calls raise, another cache on
    the same stream, and the plain functions, go on."""
    bad, good = caches(2)
    kn = rnd(1, 80, 2, 64, seed=1)
    bad.append(kn, kn, i32([0, 80]))  # five pages of three
    torch.cuda.synchronize()
    good.append(kn[:, :40], kn[:, :40], i32([0, 40]))
    q, cu, parents = rnd(3, 4, 64, seed=2), i32([0, 3]), i32([-1, 0, 1])
    good.tree_attention(0, q, kn[0, :3], kn[0, :3], parents, cu)
    paged.copy_pages(good.k, good.v, i32([0]), i32([2]))
    for call in (lambda: bad.append(kn[:, :2], kn[:, :2], i32([0, 2])), lambda: bad.free([0]), lambda: bad.compact(),
                 lambda: bad.tree_attention(0, q, kn[0, :3], kn[0, :3], parents, cu),
                 lambda: bad.prompt_attention(0, q, kn[0, :3], kn[0, :3], cu)):
        with pytest.raises(RuntimeError, match="free pages"):
            call()
    assert good.status() == 0 and paged.status("cuda:0") == 0
    assert bad.status() == _lib.ST_NO_PAGES and bad.status() == 0
    bad.append(kn[:, :2], kn[:, :2], i32([0, 2]))
    assert bad.seq_lens.tolist() == [2, 0] and good.seq_lens.tolist() == [40, 0] and bad.status() == 0


def test_a_caches_status_holds_on_every_stream():
    bad, _ = caches(2)
    kn = rnd(1, 80, 2, 64, seed=1)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bad.append(kn, kn, i32([0, 80]))
        s.synchronize()
    with pytest.raises(RuntimeError, match="free pages"):
        bad.free([0])
    assert bad.status() == _lib.ST_NO_PAGES


def test_cache_status_tells_of_attention():
    cache, _ = caches(2)
    kn, q = rnd(1, 3, 2, 64, seed=1), rnd(3, 4, 64, seed=2)
    prompt.status("cuda:0")
    cache.tree_attention(0, q, kn[0], kn[0], i32([-1, 2, 0]), i32([0, 3]))
    assert cache.status() == _lib.ST_BAD_PARENT
    cache.tree_attention(0, q, kn[0], kn[0], i32([-1, 0, 0]), i32([0, 3]))
    assert cache.status() == 0


def test_a_cache_can_be_captured_at_once():
    """Its workspace is there with it: the first call may be a captured one."""
    cache, _ = caches(2)
    kn, cu = rnd(1, 20, 2, 64, seed=1), i32([0, 20])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(kn, kn, cu)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert cache.seq_lens.tolist() == [40, 0] and cache.status() == 0
    graph.replay()  # 60 tokens need a fourth page
    assert cache.status() == _lib.ST_NO_PAGES and cache.seq_lens.tolist() == [40, 0]
    del graph
