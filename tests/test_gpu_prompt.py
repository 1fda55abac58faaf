"""prompt_attention and tree_attention against a plain 64-bit implementation."""
import math

import pytest
import torch

from adakv_b200 import _lib
from adakv_b200.prompt import prompt_attention, tree_attention
from tests.extend_cases import Case

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def ws_status():
    dev = torch.device("cuda", torch.cuda.current_device())
    return _lib.read_status(_lib.workspace(256, dev, "extend"))


def run(c, **kw):
    d = c.device
    q, k, v = c.q.to(d), c.k.to(d), c.v.to(d)
    pages = c.pages()
    slots = c.slots.int().to(d)
    if c.parents is not None:
        return tree_attention(q, k, v, c.parents.to(d), c.cu_tensor(), *pages, slots=slots,
                              return_lse=True, **kw)
    if sum(c.prefix):
        return prompt_attention(q, k, v, c.cu_tensor(), pages, slots=slots, return_lse=True, **kw)
    return prompt_attention(q, k, v, c.cu_tensor(), return_lse=True, **kw)


PROMPTS = [
    ([1], [0]), ([2, 0, 1], [0, 0, 0]), ([17], [0]), ([63, 64, 65], [0] * 3), ([127, 128, 129], [0] * 3),
    ([300, 5, 0, 700, 33], [0] * 5), ([1, 40], [1, 257]), ([200, 3, 130], [15, 1000, 0]),
    ([257], [129]), ([0, 0, 9, 0], [3, 0, 128, 0]),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", PROMPTS, ids=lambda x: f"{x[0]}+{x[1]}".replace(" ", ""))
def test_prompt(dtype, D, lens):
    c = Case(*lens, 8, 2, D, dtype, seed=len(lens[0]) + D)
    c.check(*run(c))
    assert ws_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (6, 1), (10, 2), (14, 2), (16, 1), (24, 8), (64, 1), (33, 1)])
def test_prompt_head_groups(dtype, Hq, Hkv):
    c = Case([70, 1, 131], [20, 0, 300], Hq, Hkv, 64, dtype, page=32, seed=Hq)
    c.check(*run(c))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [
    ([1], [1]), ([1], [0]), ([1], [16]), ([1, 1, 1], [5, 4000, 129]), ([8], [1000]), ([32, 6, 0, 25], [777, 0, 5, 128]),
    ([64], [1025]), ([100, 2], [63, 2048]), ([130, 260], [31, 127]),
], ids=lambda x: f"{x[0]}+{x[1]}".replace(" ", ""))
def test_tree(dtype, D, lens):
    c = Case(*lens, 8, 2, D, dtype, tree=True, seed=sum(lens[0]))
    c.check(*run(c))
    assert ws_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,tree,lens", [
    (64, True, ([1], [60000])), (128, True, ([1], [40000])), (128, True, ([12, 1], [50001, 33000])),
    (64, False, ([20], [50000])), (128, False, ([150], [30000])), (128, True, ([40], [33333])),
], ids=lambda x: str(x).replace(" ", ""))
def test_long_contexts(dtype, D, tree, lens):
    """Many key tiles to a CTA."""
    c = Case(*lens, 8, 2, D, dtype, tree=tree, seed=sum(lens[0]))
    c.check(*run(c))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("new", [[64], [65], [128], [129], [1] * 60, [3, 0, 50, 11], [127, 1], [63, 1, 1]])
def test_short_prompts_many_heads(dtype, new):
    """No more tokens than a key tile (where nothing is split), and just above,
    with more row tiles than the grid has CTAs."""
    c = Case(new, [0] * len(new), 96, 24, 64, dtype, seed=len(new) + sum(new))
    c.check(*run(c))
    assert ws_status() == 0


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_page_sizes(page, dtype):
    c = Case([3, 150, 1], [page * 3, page * 9 - 1, page + 1], 12, 2, 128, dtype, page=page, seed=page)
    c.check(*run(c))
    c = Case([3, 15, 1], [page * 30, page * 9 - 1, page + 1], 12, 2, 64, dtype, page=page, tree=True, seed=page)
    c.check(*run(c))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_sequences(dtype):
    g = torch.Generator().manual_seed(5)
    B = 150  # more than the lanes of a warp several times over, some without new tokens
    new = [int(x) for x in torch.randint(0, 9, (B,), generator=g)]
    pre = [int(x) for x in torch.randint(0, 90, (B,), generator=g)]
    c = Case(new, pre, 4, 2, 64, dtype, tree=True, seed=7)
    c.check(*run(c))
    c = Case(new, pre, 4, 2, 64, dtype, seed=8)
    c.check(*run(c))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_chain_is_causal(dtype):
    """A tree in which every token follows the one before it is the causal form."""
    c = Case([90, 7], [33, 300], 8, 2, 128, dtype, seed=3)
    a, la = run(c)
    t = Case([90, 7], [33, 300], 8, 2, 128, dtype, seed=3)
    t.parents = torch.cat([torch.arange(n) - 1 for n in t.new]).int()
    t.live[:] = True
    b, lb = run(t)
    t.check(b, lb)
    assert torch.equal(la, lb) and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tree", [False, True])
def test_strides_and_foreign_memory(dtype, tree):
    """q / k / v cut out of one projection, head-major outputs, pages of a pool
    of several layers, and NaN in all that lies between."""
    c = Case([37, 0, 130], [50, 16, 700], 8, 2, 64, dtype, tree=tree, seed=11, gap=5)
    d = "cuda"
    W = (c.Hq + 2 * c.Hkv) * c.D + 16
    proj = torch.full((c.T, W), math.nan, dtype=dtype, device=d)
    at = [0, c.Hq * c.D, (c.Hq + c.Hkv) * c.D]
    views = []
    for t, o in zip((c.q, c.k, c.v), at):
        x = proj[:, o:o + t.shape[1] * c.D].unflatten(1, (t.shape[1], c.D))
        x.copy_(t)
        views.append(x)
    kp, vp, table, lens = c.pages()
    big = torch.full((kp.shape[0], 3, *kp.shape[1:]), math.nan, dtype=dtype, device=d)
    big[:, 1], big[:, 2] = kp, vp
    wide = torch.full((table.shape[0], table.shape[1] + 7), 2 ** 30, dtype=torch.int32, device=d)
    wide[:, :table.shape[1]] = table
    out = torch.full((c.Hq, c.T, c.D), 7.0, dtype=dtype, device=d).transpose(0, 1)
    pages = (big[:, 1], big[:, 2], wide[:, :table.shape[1]], lens)
    slots = c.slots.int().to(d)
    if tree:
        o, lse = tree_attention(*views, c.parents.to(d), c.cu_tensor(), *pages, slots=slots, out=out, return_lse=True)
    else:
        o, lse = prompt_attention(*views, c.cu_tensor(), pages, slots=slots, out=out, return_lse=True)
    assert o is out
    c.check(o, lse)
    # rows of no sequence are not written
    assert (out[:5] == 7).all() and (out[-5:] == 7).all()
    assert ws_status() == 0


def test_one_layer_of_head_major_cache():
    """The framework's contiguous cache [B, Hkv, S, D] read in place as pages."""
    B, H, S, D, ps = 2, 2, 96, 64, 16
    g = torch.Generator().manual_seed(1)
    K, V = (torch.randn(B, H, S, D, generator=g).to(BF16) for _ in range(2))
    c = Case([5, 9], [90, 33], 4, H, D, BF16, seed=2, shuffle=False)
    # page j of sequence b starts (b H S + j ps) rows into the buffer; a head is S rows on
    per = H * S // ps
    table = torch.tensor([[b * per + j for j in range(S // ps)] for b in range(B)], dtype=torch.int32)
    kd, vd = K.cuda(), V.cuda()

    def paged(x):
        return x.as_strided(((B - 1) * per + S // ps, H, ps, D), (ps * D, S * D, D, 1))

    out, lse = prompt_attention(c.q.cuda(), c.k.cuda(), c.v.cuda(), c.cu_tensor(),
                                (paged(kd), paged(vd), table.cuda(), torch.tensor([90, 33], dtype=torch.int32).cuda()),
                                return_lse=True)
    # the same keys in the reference's pages
    for b in range(B):
        for j in range(-(-c.prefix[b] // ps)):
            m = min(ps, c.prefix[b] - j * ps)
            c.kp[c.table[b, j], :, :m] = K[b, :, j * ps:j * ps + m]
            c.vp[c.table[b, j], :, :m] = V[b, :, j * ps:j * ps + m]
    c.check(out, lse)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_extreme_scores(dtype):
    """Scores far apart: rows whose first key tiles weigh nothing, maxima that
    rise late, and large negative scores alone."""
    c = Case([140, 3], [400, 600], 4, 1, 64, dtype, seed=21, gain=1.0)
    ids = c.table[c.slots[0], :25].long()
    c.kp[ids[20], 0, 3] *= 60.0        # one key far above the others, late
    c.k[c.cu[0] + 100:c.cu[0] + 104] *= 40.0
    c.q[c.cu[1]:c.cu[2]] = -40.0       # all scores of the second sequence are very negative
    ids = c.table[c.slots[1], :38].long()
    c.kp[ids] = c.kp[ids].abs() + 1.0
    c.k[c.cu[1]:c.cu[2]] = c.k[c.cu[1]:c.cu[2]].abs() + 1.0
    c.check(*run(c))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_type_maximum_keys(dtype):
    """A key whose scores overflow to -inf weighs nothing, like a masked one."""
    c = Case([9], [40], 2, 1, 64, dtype, seed=4)
    c.q[:] = c.q.abs().clamp(min=0.5)
    page = c.table[c.slots[0], 1].item()
    big = torch.finfo(torch.float32).max if dtype == F32 else torch.finfo(dtype).max
    c.kp[page, 0, 2] = -big
    out, lse = run(c)
    # the same with that key far below every other
    c.kp[page, 0, 2] = -1e4
    c.check(out, lse)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_other_streams_and_graphs(dtype):
    c = Case([33, 1], [100, 333], 8, 2, 128, dtype, tree=True, seed=9)
    want, wl = run(c)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, gl = run(c)
        s.synchronize()
        assert torch.equal(got, want) and torch.equal(gl, wl)
        d = c.device
        args = [c.q.to(d), c.k.to(d), c.v.to(d), c.parents.to(d), c.cu_tensor(), *c.pages()]
        slots = c.slots.int().to(d)
        graph = torch.cuda.CUDAGraph()
        s.synchronize()
        with torch.cuda.graph(graph, stream=s):
            o, l = tree_attention(*args, slots=slots, return_lse=True)
        for _ in range(3):
            o.zero_()
            graph.replay()
            s.synchronize()
            assert torch.equal(o, want) and torch.equal(l, wl)
        # the graph reads lengths on the device: another context, same shapes
        args[8].sub_(7)
        graph.replay()
        o2, l2 = tree_attention(*args, slots=slots, return_lse=True)
        s.synchronize()
        assert torch.equal(o, o2) and torch.equal(l, l2)
    del graph


def test_repeated_calls_are_equal():
    c = Case([300, 40], [1000, 90], 8, 2, 128, BF16, seed=13)
    a, la = run(c)
    for _ in range(5):
        b, lb = run(c)
        assert torch.equal(a, b) and torch.equal(la, lb)


def test_offsets_beyond_32_bits():
    """Pages whose elements lie past 2^32 bytes and 2^31 elements of the pool."""
    ps, D = 16, 128
    n_pages = (2 ** 31) // (ps * D) + 64
    kp = torch.empty((n_pages, 1, ps, D), dtype=BF16, device="cuda")
    vp = torch.empty((n_pages, 1, ps, D), dtype=BF16, device="cuda")
    c = Case([4], [60], 4, 1, D, BF16, seed=31, shuffle=False)
    high = torch.tensor([n_pages - 1, n_pages - 3, n_pages - 64, n_pages - 7])
    old = c.table[0, :4].long()
    kp[high.cuda()] = c.kp[old].cuda()
    vp[high.cuda()] = c.vp[old].cuda()
    table = c.table.clone()
    table[0, :4] = high.int()
    out, lse = prompt_attention(c.q.cuda(), c.k.cuda(), c.v.cuda(), c.cu_tensor(),
                                (kp, vp, table.cuda(), c.lens.cuda()), return_lse=True)
    c.check(out, lse)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_values_are_reported(dtype):
    """Lengths, slots, page ids and parents out of range: no fault, a status bit,
    and the next call raises."""
    c = Case([4, 3], [30, 20], 4, 2, 64, dtype, tree=True, seed=17)
    d = c.device
    base = dict(q=c.q.to(d), k=c.k.to(d), v=c.v.to(d), parents=c.parents.to(d), cu=c.cu_tensor())
    kp, vp, table, lens = c.pages()
    slots = c.slots.int().to(d)

    def call(parents=base["parents"], cu=base["cu"], table=table, lens=lens, slots=slots):
        return tree_attention(base["q"], base["k"], base["v"], parents, cu, kp, vp, table, lens, slots=slots)

    assert ws_status() == 0
    wrong = table.clone()
    wrong[slots[0].long(), 0] = 10 ** 6
    call(table=wrong)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="page id"):
        call()
    assert ws_status() == _lib.ST_BAD_BLOCK_ID
    long = lens.clone()
    long[slots[1].long()] = 10 ** 6
    call(lens=long)
    assert ws_status() & _lib.ST_BAD_SEQ_LEN
    call(slots=torch.tensor([0, 99], dtype=torch.int32, device=d))
    assert ws_status() & _lib.ST_BAD_SEQ_LEN
    call(cu=torch.tensor([0, 400, 7], dtype=torch.int32, device=d))
    assert ws_status() & _lib.ST_BAD_SEQ_LEN
    par = base["parents"].clone()
    par[2] = 3
    call(parents=par)
    assert ws_status() & _lib.ST_BAD_PARENT
    c.check(*run(c))


def test_empty_calls():
    q = torch.empty((0, 4, 64), dtype=BF16, device="cuda")
    k = torch.empty((0, 2, 64), dtype=BF16, device="cuda")
    out, lse = prompt_attention(q, k, k, torch.zeros(3, dtype=torch.int32, device="cuda"), return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    c = Case([0, 0], [5, 6], 4, 2, 64, BF16, gap=3)
    out = torch.full((6, 4, 64), 3.0, dtype=BF16, device="cuda")
    run(c, out=out)
    assert (out == 3).all()


def test_refusals():
    c = Case([4], [10], 4, 2, 64, BF16, tree=True)
    d = c.device
    q, k, v, par, cu = c.q.to(d), c.k.to(d), c.v.to(d), c.parents.to(d), c.cu_tensor()
    kp, vp, table, lens = c.pages()
    slots = c.slots.int().to(d)
    ok = dict(slots=slots)
    tree_attention(q, k, v, par, cu, kp, vp, table, lens, **ok)
    with pytest.raises(RuntimeError, match="CUDA"):
        prompt_attention(q.cpu(), k.cpu(), v.cpu(), cu.cpu())
    for bad, text in [
        (dict(q=q[:, :, :32]), "k must"), (dict(k=k.float()), "k must"), (dict(v=v[:2]), "v must"),
        (dict(q=q[:, :3]), "multiple"), (dict(par=par.long()), "parents"), (dict(par=par[:2]), "parents"),
        (dict(cu=cu.long()), "cu_seqlens"), (dict(kp=kp[:, :1]), "k_pages"), (dict(vp=vp.half()), "v_pages"),
        (dict(table=table.long()), "page_table"), (dict(lens=lens[:1]), "seq_lens"),
        (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), "contiguous"),
        (dict(par=None), "parents"),
    ]:
        a = dict(q=q, k=k, v=v, par=par, cu=cu, kp=kp, vp=vp, table=table, lens=lens) | bad
        with pytest.raises(ValueError, match=text):
            tree_attention(*a.values(), **ok)
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)):
        with pytest.raises(ValueError, match="scale"):
            tree_attention(q, k, v, par, cu, kp, vp, table, lens, **ok, **kw)
    with pytest.raises(ValueError, match="slots"):
        tree_attention(q, k, v, par, cu, kp, vp, table, lens, slots=slots.long())
    with pytest.raises(ValueError, match="slots"):
        prompt_attention(q, k, v, cu, slots=slots)
    with pytest.raises(NotImplementedError, match="head_dim"):
        z = torch.zeros((4, 4, 96), dtype=BF16, device=d)
        prompt_attention(z, z, z, cu)
    with pytest.raises(NotImplementedError, match="page_size"):
        tree_attention(q, k, v, par, cu, kp[:, :, :8], vp[:, :, :8], table, lens, **ok)
    with pytest.raises(ValueError, match="16"):  # rows off their 16-byte boundary
        flat = torch.zeros(4 * 4 * 64 + 8, dtype=BF16, device=d)
        prompt_attention(flat[1:1 + 4 * 4 * 64].view(4, 4, 64), k, v, cu)
    with pytest.raises(ValueError, match="stride"):  # a broadcast axis
        prompt_attention(q, k[:, :1].expand(4, 2, 64), v, cu)
    with pytest.raises(ValueError, match="dtype"):
        prompt_attention(q.double(), k.double(), v.double(), cu)
