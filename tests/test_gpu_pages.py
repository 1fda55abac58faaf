"""The paged cache's operators against a plain model that keeps every sequence's
tokens in Python lists."""
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


class Model:
    """Page table, lengths and counts as the rules say, on the host."""

    def __init__(self, n_pages, n_slots, width, ps):
        self.N, self.W, self.ps = n_pages, width, ps
        self.rows = [[] for _ in range(n_slots)]
        self.toks = [[] for _ in range(n_slots)]

    def ref(self):
        r = [0] * self.N
        for row in self.rows:
            for p in row:
                r[p] += 1
        return r

    def free_ids(self):
        return [i for i, x in enumerate(self.ref()) if x == 0]

    def fork(self, src, dst):
        free = self.free_ids()
        before = [(list(self.rows[s]), list(self.toks[s])) for s in src]  # as the call finds them
        for (row, toks), d in zip(before, dst):
            if len(toks) % self.ps:
                row[-1] = free.pop(0)
            self.rows[d], self.toks[d] = row, toks

    def free(self, slots):
        for s in slots:
            self.rows[s], self.toks[s] = [], []

    def append(self, slots, toks):
        free = self.free_ids()
        for s, t in zip(slots, toks):
            self.toks[s] += t
            while len(self.rows[s]) * self.ps < len(self.toks[s]):
                self.rows[s].append(free.pop(0))

    def compact(self):
        ref = self.ref()
        live = sum(x > 0 for x in ref)
        movers = [i for i in range(live, self.N) if ref[i]]
        holes = [i for i in range(live) if not ref[i]]
        to = dict(zip(movers, holes))
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]

    def check(self, c):
        table = torch.full((len(self.rows), self.W), -1, dtype=torch.int32)
        for s, row in enumerate(self.rows):
            table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
        assert torch.equal(c.page_table.cpu(), table)
        assert c.seq_lens.tolist() == [len(t) for t in self.toks]
        assert c.refcounts.tolist() == self.ref()
        k, v = c.k.cpu(), c.v.cpu()
        for row, toks in zip(self.rows, self.toks):
            for j, t in enumerate(toks):
                at = (slice(None), row[j // self.ps], slice(None), j % self.ps)
                assert torch.equal(k[at], token(t, c.k)) and torch.equal(v[at], -token(t, c.k))


def token(t, like):
    """The k rows of token number t, [layers, heads, head_dim]."""
    L, _, H, _, D = like.shape
    base = torch.arange(L * H * D, dtype=torch.float32).reshape(L, H, D)
    return ((base * 7 + t * 13) % 251 - 125).to(like.dtype)


def tokens(ts, like):
    x = torch.stack([token(t, like) for t in ts], 1).to(like.device)
    return x, -x


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("L,H,D,ps", [(1, 1, 64, 16), (3, 2, 128, 16), (2, 5, 64, 32), (1, 8, 128, 128)])
def test_random_histories(dtype, L, H, D, ps):
    g = torch.Generator().manual_seed(L * 100 + H)

    def rand(n):
        return int(torch.randint(0, n, (1,), generator=g))

    N, S, maxlen = 90, 12, 5 * ps
    c = PagedKVCache(L, N, H, D, ps, S, maxlen, dtype, "cuda")
    m = Model(N, S, c.max_pages, ps)
    m.check(c)
    number = 0
    for step in range(40):
        op = rand(5)
        empty = [s for s in range(S) if not m.toks[s]]
        if op <= 1:  # append to some rows, by each of the three ways
            rows = torch.randperm(S, generator=g)[:1 + rand(S)].tolist()
            rows = [s for s in rows if len(m.toks[s]) + 20 <= maxlen]
            if not rows:
                continue
            n = [rand(21) for _ in rows]
            ts = [[number + 100 * i + j for j in range(x)] for i, x in enumerate(n)]
            number += 100 * len(rows)
            if sum(n) == 0:
                continue
            need = sum(-(-(len(m.toks[s]) + x) // ps) for s, x in zip(rows, n))
            if need > len(m.free_ids()):
                continue
            cu = [0]
            for x in n:
                cu.append(cu[-1] + x)
            k, v = tokens(sum(ts, []), c.k)
            way = rand(3)
            if way == 0:
                c.append(k, v, i32(cu), slots=i32(rows))
                took = ts
            elif way == 1:
                counts = [rand(x + 1) for x in n]
                c.append(k, v, i32(cu), slots=i32(rows), counts=i32(counts))
                took = [t[:x] for t, x in zip(ts, counts)]
            else:
                picks = [sorted(torch.randperm(x, generator=g)[:rand(x + 1)].tolist()) for x in n]
                wide = max(1, max(len(p) for p in picks))
                index = [p + [0] * (wide - len(p)) for p in picks]
                c.append(k, v, i32(cu), slots=i32(rows), index=i32(index),
                         counts=i32([len(p) for p in picks]))
                took = [[t[i] for i in p] for t, p in zip(ts, picks)]
            m.append(rows, took)
        elif op == 2 and empty:
            dst = empty[:1 + rand(len(empty))]
            src = [rand(S) for _ in dst]
            src = [s if s not in dst else dst[0] for s in src]  # (an empty row forks as one)
            if sum(len(m.toks[s]) % ps > 0 for s in src) > len(m.free_ids()):
                continue
            c.fork(src, dst)
            m.fork(src, dst)
        elif op == 3:
            rows = [rand(S) for _ in range(1 + rand(4))]  # some twice
            c.free(rows)
            m.free(rows)
        elif op == 4:
            c.compact()
            m.compact()
        assert c.status() == 0
        if step % 4 == 3:
            m.check(c)
    m.check(c)


@pytest.mark.parametrize("H,ps,D,dtype", [(1, 16, 64, torch.bfloat16), (8, 16, 128, torch.bfloat16),
                                          (3, 32, 128, torch.float32), (16, 128, 128, torch.float16)])
def test_copy(H, ps, D, dtype):
    pool = torch.randn(2, 2, 20, H, ps, D, device="cuda").to(dtype)
    k, v = pool[:, 0], pool[:, 1]  # strided layers
    kc, vc = k.clone(), v.clone()
    src, dst = i32([3, 0, 19, 3]), i32([7, 18, 1, 2])
    paged.copy_pages(k, v, src, dst)
    kc[:, dst.long()] = kc[:, src.long()]
    vc[:, dst.long()] = vc[:, src.long()]
    assert torch.equal(k, kc) and torch.equal(v, vc)
    paged.copy_pages(k, v, i32([]), i32([]))
    paged.copy_pages(k, v, i32([4, -1, 5]), i32([6, 8, 20]))  # bad ids are skipped
    kc[:, 6], vc[:, 6] = kc[:, 4], vc[:, 4]
    assert torch.equal(k, kc) and torch.equal(v, vc)
    assert paged.status(k.device) == _lib.ST_BAD_BLOCK_ID


def test_large_pool():
    """More pages than one pass of the plan reads, with the free ones at the end
    and holes throughout."""
    N, ps = 50000, 16
    c = PagedKVCache(1, N, 1, 64, ps, 8, N * ps, torch.bfloat16, "cuda")
    c.k.normal_()
    c.v.normal_()
    held = [20000, 9000, 15000]
    order = torch.randperm(45000, generator=torch.Generator().manual_seed(1)).int()
    at = 0
    for s, n in enumerate(held):
        c.page_table[s, :n] = order[at:at + n].cuda()
        c.seq_lens[s] = n * ps
        at += n
    c.refcounts[order[:at].long().cuda()] = 1
    want = [c.k[0, c.page_table[s, :n].long()].clone() for s, n in enumerate(held)]
    c.free([1])
    c.compact()
    assert c.status() == 0
    live = held[0] + held[2]
    ref = c.refcounts
    assert (ref[:live] == 1).all() and (ref[live:] == 0).all()
    for s in (0, 2):
        ids = c.page_table[s, :held[s]].long()
        assert (ids < live).all() and torch.equal(c.k[0, ids], want[s])
        assert ids.unique().numel() == held[s]
    k = torch.randn(1, 40, 1, 64, device="cuda").to(torch.bfloat16)
    c.append(k, k, i32([0, 40]), slots=i32([5]))
    assert c.page_table[5, :4].tolist() == [live, live + 1, live + 2, -1]
    assert c.status() == 0


def fresh():
    c = PagedKVCache(2, 6, 2, 64, 16, 5, 64, torch.bfloat16, "cuda")
    m = Model(6, 5, c.max_pages, 16)
    k, v = tokens(list(range(40)), c.k)
    c.append(k, v, i32([0, 40]), slots=i32([1]))
    m.append([1], [list(range(40))])
    return c, m


@pytest.mark.parametrize("call,bits", [
    (lambda c, k: c.fork([1, 1, 1, 1], [0, 2, 3, 4]), _lib.ST_NO_PAGES),
    (lambda c, k: c.fork([1, 1], [0, 0]), _lib.ST_BAD_SLOT),
    (lambda c, k: c.fork([0], [1]), _lib.ST_BAD_SLOT),
    (lambda c, k: c.fork([5], [0]), _lib.ST_BAD_SLOT),
    (lambda c, k: c.fork([1], [-1]), _lib.ST_BAD_SLOT),
    (lambda c, k: c.append(k, k, i32([0, 40, 80]), slots=i32([0, 1])), _lib.ST_BAD_SEQ_LEN),
    (lambda c, k: c.append(k, k, i32([0, 64]), slots=i32([0])), _lib.ST_NO_PAGES),
    (lambda c, k: c.append(k, k, i32([0, 5, 9]), slots=i32([0, 0])), _lib.ST_BAD_SLOT),
    (lambda c, k: c.append(k, k, i32([0, 5]), slots=i32([7])), _lib.ST_BAD_SLOT),
    (lambda c, k: c.append(k, k, i32([0, 5]), counts=i32([6])), _lib.ST_BAD_SEQ_LEN),
    (lambda c, k: c.append(k, k, i32([0, 5]), counts=i32([-1])), _lib.ST_BAD_SEQ_LEN),
    (lambda c, k: c.append(k, k, i32([3, 90])), _lib.ST_BAD_SEQ_LEN),
    (lambda c, k: c.append(k, k, i32([5, 3])), _lib.ST_BAD_SEQ_LEN),
    (lambda c, k: c.append(k, k, i32([0, 5]), index=i32([[0, 5]]), counts=i32([2])), _lib.ST_BAD_SEQ_LEN),
], ids=range(14))
def test_requests_that_cannot_be_met_change_nothing(call, bits):
    c, m = fresh()
    k = torch.ones(2, 80, 2, 64, dtype=torch.bfloat16, device="cuda")
    if bits == _lib.ST_NO_PAGES and "fork" not in call.__code__.co_names:
        c.fork([1], [2])  # leaves two free pages
        m.fork([1], [2])
    call(c, k)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="status"):
        c.free([0])
    assert c.status() & bits
    m.check(c)
    c.free([0])
    assert c.status() == 0


def test_bad_rows_of_free():
    c, m = fresh()
    c.free([-1, 9, 1])
    m.free([1])
    assert c.status() == _lib.ST_BAD_SLOT
    m.check(c)


def test_graph_of_page_calls():
    c, m = fresh()
    k, v = tokens(list(range(100, 103)), c.k)
    cu, slots = i32([0, 3]), i32([2])
    src, dst = i32([1]), i32([2])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.fork(src, dst)  # makes the stream's workspace
        c.free(dst)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.fork(src, dst)
            c.append(k, v, cu, slots=slots)
            c.compact()
            c.free(src)
            c.compact()
        g.replay()
        s.synchronize()
        assert c.status() == 0
    m.fork([1], [2])
    m.append([2], [[100, 101, 102]])
    m.compact()
    m.free([1])
    m.compact()
    m.check(c)
    del g


def test_refusals():
    c, _ = fresh()
    k = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device="cuda")
    cu = i32([0, 4])
    with pytest.raises(ValueError, match="src"):
        c.copy(torch.zeros(2, dtype=torch.int64, device="cuda"), i32([0, 1]))
    with pytest.raises(ValueError, match="dst"):
        c.fork(i32([0, 1]), i32([2]))
    with pytest.raises(ValueError, match="slots"):
        c.free(torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="k_new"):
        c.append(k[:1], k[:1], cu)
    with pytest.raises(ValueError, match="v_new"):
        c.append(k, k.float(), cu)
    with pytest.raises(ValueError, match="one shape"):
        c.append(k, k[:, :2], cu)
    with pytest.raises(ValueError, match="index"):
        c.append(k, k, cu, index=i32([0, 1]))
    with pytest.raises(ValueError, match="counts"):
        c.append(k, k, cu, counts=i32([1, 1]))
    with pytest.raises(ValueError, match="contiguous"):
        paged.copy_pages(c.k.transpose(2, 3), c.v.transpose(2, 3), i32([0]), i32([1]))
    with pytest.raises(ValueError, match="refcounts"):
        paged.fork_sequences(c.k, c.v, c.page_table, c.seq_lens, c.refcounts[:-1], i32([0]), i32([1]))
    with pytest.raises(ValueError, match="one shape"):
        paged.compact_pages(c.k, c.v[:1], c.page_table, c.seq_lens, c.refcounts)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.copy_pages(c.k.cpu(), c.v.cpu(), i32([0]), i32([1]))
    with pytest.raises(ValueError, match="page_size"):
        PagedKVCache(1, 4, 1, 64, page_size=8)
    with pytest.raises(NotImplementedError, match="head_dim"):
        PagedKVCache(1, 4, 1, 96)
    with pytest.raises(ValueError, match="1 or more"):
        PagedKVCache(0, 4, 1, 64)
    with pytest.raises(ValueError, match="dtype"):
        PagedKVCache(1, 4, 1, 64, dtype=torch.float64)
    assert c.status() == 0
