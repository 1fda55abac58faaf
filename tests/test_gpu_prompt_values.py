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
