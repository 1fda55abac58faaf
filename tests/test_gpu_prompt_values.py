"""prompt_attention and tree_attention where values are not finite, or probabilities
too small for the element type."""
import math

import pytest
import torch

from adakv_b200.prompt import prompt_attention, tree_attention

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def pages_of(k, v, ps=16):
    """[n, Hkv, D] keys and values of one sequence as pages, table and length."""
    n, H, D = k.shape
    m = -(-n // ps)
    out = []
    for t in (k, v):
        x = torch.full((m * ps, H, D), math.nan, dtype=t.dtype, device=t.device)
        x[:n] = t
        out.append(x.view(m, ps, H, D).transpose(1, 2).contiguous())
    return (*out, torch.arange(m, dtype=torch.int32, device=k.device)[None],
            torch.tensor([n], dtype=torch.int32, device=k.device))


def rnd(*shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("new,prefix", [(5, 0), (130, 0), (3, 50), (2, 9000)])
def test_nan_query_gives_nan_lse(dtype, new, prefix):
    """A query of NaN: its row's output and log-sum-exp are NaN, whether the row
    tile is computed by one CTA or in pieces; every other row is as without it."""
    q, k, v = (rnd(new, h, 64, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    pages = pages_of(rnd(prefix, 2, 64, seed=3, dtype=dtype), rnd(prefix, 2, 64, seed=4, dtype=dtype)) if prefix else None
    cu = i32([0, new])
    want, wl = prompt_attention(q, k, v, cu, pages, return_lse=True)
    q[1, 3] = math.nan
    out, lse = prompt_attention(q, k, v, cu, pages, return_lse=True)
    assert torch.isnan(lse[1, 3]) and torch.isnan(out[1, 3]).all()
    other = torch.ones_like(lse, dtype=torch.bool)
    other[1, 3] = False
    assert torch.equal(lse[other], wl[other]) and torch.equal(out[other], want[other])
    assert torch.isfinite(wl).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("prefix", [40, 9000])
@pytest.mark.parametrize("where", ["q", "k"])
def test_infinite_scores_are_not_hidden(dtype, prefix, where):
    """A score of +inf (or NaN) makes softmax NaN: neither a finite output nor an
    lse that a merge would take for an empty or finite part."""
    q, k, v = (rnd(3, h, 64, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    kc, vc = rnd(prefix, 2, 64, seed=3, dtype=dtype), rnd(prefix, 2, 64, seed=4, dtype=dtype)
    if where == "q":
        q[2, 1, 7] = math.inf
        rows = [(2, 1)]
    else:
        q[:, :2, 7] = q[:, :2, 7].abs() + 0.5
        kc[prefix // 2, 0, 7] = math.inf
        rows = [(t, h) for t in range(3) for h in (0, 1)]
    out, lse = prompt_attention(q, k, v, i32([0, 3]), pages_of(kc, vc), return_lse=True)
    hit = torch.zeros_like(lse, dtype=torch.bool)
    for r in rows:
        hit[r] = True
    assert torch.isnan(out[hit]).all()
    assert not (lse[hit] < math.inf).any()  # NaN or +inf
    assert torch.isfinite(out[~hit]).all() and torch.isfinite(lse[~hit]).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("prefix", [40, 9000])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_unused_slots_are_zero_beside_infinite_values(dtype, prefix, value):
    """An unused tree slot sees no key: its output is 0 also where a cached value is
    infinite or NaN; the slots that see it show that in its element alone."""
    q, k, v = (rnd(4, h, 64, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    kc, vc = rnd(prefix, 2, 64, seed=3, dtype=dtype), rnd(prefix, 2, 64, seed=4, dtype=dtype)
    vc[prefix // 3, 1, 9] = value
    kp, vp, table, lens = pages_of(kc, vc)
    out, lse = tree_attention(q, k, v, i32([-1, -2, 0, -2]), i32([0, 4]), kp, vp, table, lens, return_lse=True)
    assert (out[1] == 0).all() and (out[3] == 0).all()
    assert (lse[1] == -math.inf).all() and (lse[3] == -math.inf).all()
    assert torch.isfinite(lse[0]).all() and torch.isfinite(lse[2]).all()
    for t in (0, 2):
        bad = ~torch.isfinite(out[t])
        want = torch.zeros_like(bad)
        want[2:, 9] = True  # the heads of KV head 1
        assert torch.equal(bad, want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n,B,heads", [(100, 1, 4), (3000, 1, 4), (3000, 40, 64)])
@pytest.mark.parametrize("at", [0, 1])
def test_many_small_probabilities(dtype, n, B, heads, at):
    """One key outweighs every other one 2^26 to 2^24 times but has a value of 0 (an
    attention sink): the output is what all the others add up to.

    With w the weights and the largest of them close to 1, P's rounding costs at most
    e w and, of fp16, half its smallest step 2^-24, 2^-7 of the type's steps for what
    the kernel scales up: 2^-32 a key."""
    D, Hkv = 64, heads // 4
    g = torch.Generator().manual_seed(n + B)
    kc, vc = torch.zeros(n, Hkv, D), 300.0 + 200.0 * torch.rand((n, Hkv, D), generator=g)
    kc[:, :, 0] = -(17.3 + 0.7 * torch.rand((n, Hkv), generator=g)) / 2  # scores, with q = 16
    sink = (n - 1) * at
    kc[sink], vc[sink] = 0, 0
    kc, vc = kc.to(dtype).cuda(), vc.to(dtype).cuda()
    q, kn, vn = torch.zeros(B, heads, D), torch.zeros(B, Hkv, D), torch.zeros(B, Hkv, D)
    q[:, :, 0], kn[:, :, 0] = 16.0, -9.0
    kp, vp, table, lens = pages_of(kc, vc)
    out, lse = tree_attention(q.to(dtype).cuda(), kn.to(dtype).cuda(), vn.to(dtype).cuda(), i32([-1] * B),
                              torch.arange(B + 1, dtype=torch.int32, device="cuda"), kp, vp, table.repeat(B, 1),
                              lens.repeat(B), return_lse=True)
    z = torch.cat([kc[:, :, 0].double().cpu() * 2, torch.full((1, Hkv), -18.0)])  # [n + 1, Hkv]
    v = torch.cat([vc.double().cpu(), torch.zeros(1, Hkv, D)])
    w = torch.softmax(z, 0)
    want = torch.einsum("nh,nhd->hd", w, v).repeat_interleave(4, 0)
    u, e = 2.0 ** -22, {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}[dtype]
    tol = want * (2 * e + (n + 16) * u + 2 * 18 * (D + 4) * u)
    if dtype == F16:
        tol = tol + v.sum(0).repeat_interleave(4, 0) * 2.0 ** -32 + 2.0 ** -25
    assert ((out.double().cpu() - want).abs() <= tol).all()
    L = torch.logsumexp(z, 0).repeat_interleave(4, 0)
    assert ((lse.double().cpu() - L).abs() <= (18 * (D + 4) + n + 16) * u).all()


def outcome(vis, v, clean):
    """[T, Hq, D] outputs where the new tokens' v [T, Hkv, D] holds values that are not
    finite: `clean` (with 0 in their place) and, for the rows that see them (vis [T, T]),
    their sum."""
    bad = torch.where(torch.isfinite(v), 0.0, v.double())
    add = torch.zeros(clean.shape, dtype=torch.float64, device=v.device)
    for j in torch.nonzero(~torch.isfinite(v).all(-1).all(-1))[:, 0].tolist():
        add += torch.where(vis[:, j, None, None], bad[j].repeat_interleave(clean.shape[1] // v.shape[1], 0)[None], 0.0)
    return clean.double() + add


def same(a, b):
    return ((a.double() == b) | (torch.isnan(a) & torch.isnan(b))).all()


def spoil(v, at, seed):
    """Infinities and NaN in a few elements of the tokens `at`."""
    g = torch.Generator().manual_seed(seed)
    for t in at:
        for _ in range(3):
            h, d = (int(torch.randint(0, n, (1,), generator=g)) for n in v.shape[1:])
            v[t, h, d] = (math.inf, -math.inf, math.nan)[int(torch.randint(0, 3, (1,), generator=g))]
    return v


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (6, 2), (64, 1)])
@pytest.mark.parametrize("n,prefix,at", [(7, 0, [3, 6]), (200, 0, [0, 63, 64, 130, 199]), (150, 9000, [20, 149]),
                                         (700, 33, [5, 300, 301, 640])])
def test_infinite_values_of_later_tokens_stay_out(dtype, D, Hq, Hkv, n, prefix, at):
    """V of a prompt's later tokens may be infinite or NaN: rows before them are bit
    for bit as without, the rows from them on have it in its element alone."""
    q, k, v = (rnd(n, h, D, seed=i, dtype=dtype) for i, h in enumerate((Hq, Hkv, Hkv)))
    pages = pages_of(rnd(prefix, Hkv, D, seed=3, dtype=dtype), rnd(prefix, Hkv, D, seed=4, dtype=dtype)) if prefix else None
    cu = i32([0, n])
    v = spoil(v, at, n + D)
    clean, cl = prompt_attention(q, k, torch.where(torch.isfinite(v), v, 0), cu, pages, return_lse=True)
    out, lse = prompt_attention(q, k, v, cu, pages, return_lse=True)
    vis = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    assert torch.isfinite(clean).all() and torch.equal(lse, cl)
    assert same(out, outcome(vis, v, clean))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (10, 2)])
@pytest.mark.parametrize("new,prefix", [([6], 40), ([30, 1, 64], 500), ([150, 2], 20), ([90], 9000)])
def test_infinite_values_of_other_branches_stay_out(dtype, D, Hq, Hkv, new, prefix):
    """The same for drafted trees: a branch's infinite value is its own affair."""
    T, B = sum(new), len(new)
    q, k, v = (rnd(T, h, D, seed=i, dtype=dtype) for i, h in enumerate((Hq, Hkv, Hkv)))
    kp, vp, table, lens = pages_of(rnd(prefix, Hkv, D, seed=3, dtype=dtype), rnd(prefix, Hkv, D, seed=4, dtype=dtype))
    table, lens = table.repeat(B, 1), lens.repeat(B)
    g = torch.Generator().manual_seed(T)
    cu, parents, vis = [0], [], torch.zeros(T, T, dtype=torch.bool)
    for n in new:
        for i in range(n):
            parents.append(-2 if i % 11 == 10 else max(-1, i - 1 - int(torch.randint(0, 4, (1,), generator=g))))
        at = cu[-1]
        for i in range(n):
            j = i
            while j >= 0 and parents[at + j] >= -1:
                vis[at + i, at + j] = True
                j = parents[at + j]
        cu.append(at + n)
    v = spoil(v, sorted({0, T // 3, T // 2, T - 1}), T + D)
    args = (i32(parents), i32(cu), kp, vp, table, lens)
    clean, cl = tree_attention(q, k, torch.where(torch.isfinite(v), v, 0), *args, return_lse=True)
    out, lse = tree_attention(q, k, v, *args, return_lse=True)
    assert torch.isfinite(clean).all() and torch.equal(lse, cl)
    assert same(out, outcome(vis.cuda(), v, clean))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tree", [False, True])
def test_infinite_keys_of_unseen_tokens_stay_out(dtype, tree):
    """K of a later token, or of another branch, may be infinite or NaN: the rows that
    do not see it are bit for bit as without; of those that do, no output is finite."""
    n = 90
    q, k, v = (rnd(n, h, 64, seed=i, dtype=dtype) for i, h in enumerate((4, 2, 2)))
    kc, vc = rnd(50, 2, 64, seed=3, dtype=dtype), rnd(50, 2, 64, seed=4, dtype=dtype)
    pages = pages_of(kc, vc)
    parents = [i - 1 if not tree or i % 3 else i - 3 for i in range(n)]  # tree: a trunk with twigs
    parents = [max(p, -1) for p in parents]
    vis = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        j = i
        while j >= 0:
            vis[i, j] = True
            j = parents[j]
    bad = k.clone()
    bad[40, 1, 3], bad[41, 1, 7], bad[71, 1] = math.nan, math.inf, -math.inf

    def call(k):
        if tree:
            return tree_attention(q, k, v, i32(parents), i32([0, n]), *pages, return_lse=True)
        return prompt_attention(q, k, v, i32([0, n]), pages, return_lse=True)

    want, wl = call(k)
    out, lse = call(bad)
    sees = vis[:, 40].cuda()  # (NaN whatever the query is)
    free = ~(vis[:, 40] | vis[:, 41] | vis[:, 71]).cuda()
    assert free.sum() >= 40 and sees.any()
    assert torch.equal(out[free], want[free]) and torch.equal(lse[free], wl[free])
    assert torch.equal(out[:, :2], want[:, :2]) and torch.equal(lse[:, :2], wl[:, :2])  # KV head 0
    assert torch.isnan(out[sees, 2:]).all() and not (lse[sees, 2:] < math.inf).any()
