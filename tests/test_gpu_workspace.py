"""Graphs of attention and page calls, and errors that they report, when later calls
on the stream need larger workspaces."""
import pytest
import torch

from adakv_b200 import _lib, paged
from adakv_b200.prompt import tree_attention

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


def drafted(D, dtype=torch.bfloat16):
    """Arguments of a tree over a context long enough to be split."""
    n = 6000
    kp, vp = rnd(n // 16, 2, 16, D, seed=1, dtype=dtype), rnd(n // 16, 2, 16, D, seed=2, dtype=dtype)
    table = torch.arange(n // 16, dtype=torch.int32, device="cuda")[None]
    return (rnd(4, 8, D, seed=3, dtype=dtype), rnd(4, 2, D, seed=4, dtype=dtype), rnd(4, 2, D, seed=5, dtype=dtype),
            i32([-1, 0, 0, 1]), i32([0, 4]), kp, vp, table, i32([n - 3]))


def test_graph_outlives_growth():
    """A graph of a small model's calls, replayed after the same stream has served a
    larger model and a larger pool: right, and nobody else's memory is written."""
    s = torch.cuda.Stream()  # (a stream whose workspaces are not yet large)
    for key in [k for k in _lib._workspaces if k[1] == s.cuda_stream and k[2] in ("extend", "pages")]:
        _lib._workspaces.pop(key)
    with torch.cuda.stream(s):
        args = drafted(64)
        k, v = rnd(1, 40, 2, 16, 64, seed=6), rnd(1, 40, 2, 16, 64, seed=7)
        meta = [torch.full((4, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"),
                torch.zeros(40, dtype=torch.int32, device="cuda")]
        kn = rnd(1, 20, 2, 64, seed=8)
        cu, slots = i32([0, 20]), i32([2])

        def calls():
            o = tree_attention(*args, return_lse=True)
            paged.append_tokens(k, v, *meta, kn, kn, cu, slots=slots)
            return o

        want, wl = calls()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out, lse = calls()
        before = {kind: _lib._workspaces[s.device_index, s.cuda_stream, kind].data_ptr() for kind in ("extend", "pages")}
        # the larger model, and a pool of more pages
        tree_attention(*drafted(128))
        tree_attention(*drafted(128, torch.float32))
        big = torch.zeros((1, 60000, 1, 16, 64), dtype=torch.bfloat16, device="cuda")
        paged.copy_pages(big, big.clone(), i32([1]), i32([2]))
        for kind, at in before.items():
            assert _lib._workspaces[s.device_index, s.cuda_stream, kind].data_ptr() != at
        # whatever the allocator would give away again, as other tensors
        others = [torch.full((n,), 77, dtype=torch.uint8, device="cuda")
                  for n in (512, 50000, 60000, 1 << 20, 20 << 20, 20 << 20, 40 << 20)]
        out.zero_()
        graph.replay()
        s.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, wl)
        assert meta[1].tolist() == [0, 0, 40, 0]
        assert all(bool((x == 77).all()) for x in others)
    del graph


def test_error_outlives_growth():
    """A failure that nobody has read yet is raised by a call that needs a larger
    workspace, and one of a graph's replay with the smaller workspace as well."""
    s = torch.cuda.Stream()
    for key in [k for k in _lib._workspaces if k[1] == s.cuda_stream and k[2] == "pages"]:
        _lib._workspaces.pop(key)
    with torch.cuda.stream(s):
        k = torch.zeros((1, 4, 1, 16, 64), dtype=torch.bfloat16, device="cuda")
        big = torch.zeros((1, 60000, 1, 16, 64), dtype=torch.bfloat16, device="cuda")
        src, bad, one = i32([0]), i32([9]), i32([1])
        paged.copy_pages(k, k.clone(), src, one)
        assert paged.status("cuda:0") == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            paged.copy_pages(k, k, bad, one)
        paged.copy_pages(k, k.clone(), bad, one)
        s.synchronize()
        with pytest.raises(RuntimeError, match="page id"):
            paged.copy_pages(big, big, src, one)
        assert paged.status("cuda:0") == _lib.ST_BAD_BLOCK_ID
        paged.copy_pages(big, big, src, one)
        assert paged.status("cuda:0") == 0
        graph.replay()
        s.synchronize()
        with pytest.raises(RuntimeError, match="page id"):
            paged.copy_pages(big, big, src, one)
        assert paged.status("cuda:0") == _lib.ST_BAD_BLOCK_ID
        assert paged.status("cuda:0") == 0
    del graph


def test_threads_on_one_stream():
    """Threads that append to, fork and free sequences of pools of their own on the
    default stream, with attention in between: each finds its own pages as it left them."""
    import threading
    errors = []

    def work(seed):
        try:
            k, v = (torch.zeros((2, 60, 2, 16, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
            meta = [torch.full((8, 8), -1, dtype=torch.int32, device="cuda"),
                    torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(60, dtype=torch.int32, device="cuda")]
            kn = rnd(2, 61, 2, 64, seed=seed)
            cu = i32([0, 20 + seed, 61])
            q = rnd(61, 4, 64, seed=seed + 50)
            for _ in range(10):
                paged.append_tokens(k, v, *meta, kn, -kn, cu, slots=i32([1, 2]))
                paged.fork_sequences(k, v, *meta, i32([1, 2]), i32([3, 0]))
                parents = torch.arange(61, dtype=torch.int32, device="cuda") - 1
                parents[20 + seed:] -= 20 + seed
                a = tree_attention(q, kn[0], kn[0], parents, cu, k[0], v[0], meta[0], meta[1], slots=i32([1, 2]))
                b = tree_attention(q, kn[0], kn[0], parents, cu, k[0], v[0], meta[0], meta[1], slots=i32([3, 0]))
                assert torch.equal(a, b)
                for row, lo, hi in ((1, 0, 20 + seed), (2, 20 + seed, 61), (3, 0, 20 + seed), (0, 20 + seed, 61)):
                    ids = meta[0][row, :-(-(hi - lo) // 16)].long()
                    got = k[:, ids].transpose(2, 3).reshape(2, -1, 2, 64)[:, :hi - lo]
                    assert torch.equal(got, kn[:, lo:hi])
                paged.free_sequences(*meta, i32([0, 1, 2, 3]))
                assert int(meta[2].sum()) == 0
        except BaseException as e:  # noqa: BLE001 (reported by the main thread)
            errors.append(e)

    work(0)  # the workspaces
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert paged.status("cuda:0") == 0
