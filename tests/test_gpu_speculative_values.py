"""Speculative decoding over the paged cache in 16 bits, token by token and page by
page against a plain forward pass in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def plain(model, tokens, dtype):
    """Logits and every layer's keys and values [tokens, kv heads, dim] of one
    sequence, causal, with every operation rounded to `dtype` (the weights are the
    model's, as it rounded them)."""
    w = {n: getattr(model, n).to(dtype) for n in ("embed", "next")}
    wqkv, wo = ([x.to(dtype) for x in getattr(model, n)] for n in ("wqkv", "wo"))
    n, H, K, D = len(tokens), model.heads, model.kv_heads, model.dim
    pos = torch.arange(n, device=w["embed"].device)
    f = 10000.0 ** (-torch.arange(D // 2, device=pos.device, dtype=torch.float64) / (D // 2))
    c, s = ((pos[:, None] * f).cos()[:, None], (pos[:, None] * f).sin()[:, None])

    def rotate(x):
        lo, hi = x[..., :D // 2].double(), x[..., D // 2:].double()
        return torch.cat([lo * c - hi * s, hi * c + lo * s], -1).to(dtype)

    x = e = w["embed"][torch.tensor(tokens, device=pos.device)]
    keys, values = [], []
    mask = torch.ones(n, n, dtype=torch.bool, device=pos.device).tril()
    for a, b in zip(wqkv, wo):
        h = (x.double() * (x.double().square().mean(-1, keepdim=True) + torch.finfo(model.embed.dtype).eps).rsqrt()).to(dtype)
        q, k, v = (h @ a.T).unflatten(1, (-1, D)).split([H, K, K], 1)
        q, k = rotate(q), rotate(k)
        keys.append(k)
        values.append(v)
        q, k, v = q.transpose(0, 1), *(t.repeat_interleave(H // K, 1).transpose(0, 1) for t in (k, v))
        z = (q @ k.transpose(1, 2) / D ** 0.5).masked_fill(~mask, float("-inf"))
        o = torch.softmax(z.double(), -1).to(dtype) @ v
        x = x + o.transpose(0, 1).flatten(1) @ b.T
    return (x - e + e @ w["next"].T) @ w["embed"].T, torch.stack(keys), torch.stack(values)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("seed", [0, 1])
def test_tokens_and_pages_of_16_bit_decoding(dtype, seed):
    """Every token that a step emits is the likeliest next one of the 64-bit pass over
    the tokens before it, or as near to it as 16-bit rounding leaves open: within four
    times the largest error of the plain 16-bit pass over the same tokens (the two
    compared logits of either pass carry one each).  The cache holds, behind forks,
    accepted paths and a compaction, the keys and values of those tokens."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from adakv_b200.paged import PagedKVCache
    from examples.speculative_paged import TinyLM, prefill, speculative_step
    model = TinyLM(dtype=dtype, seed=seed)
    cache = PagedKVCache(model.n_layers, 400, model.kv_heads, model.dim, 16, n_slots=12, max_seq_len=640, dtype=dtype)
    g = torch.Generator().manual_seed(seed + 1)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (45, 160, 1)]
    slots = cache._ids([0, 1, 2])
    prefill(model, cache, [prompts[0][:20], prompts[1][:100], []], slots)
    last = prefill(model, cache, [prompts[0][20:], prompts[1][100:], prompts[2]], slots)
    cache.fork([0, 1, 2], [3, 4, 5])
    rows = cache._ids([0, 1, 2, 3, 4, 5])
    last = last + last
    seqs = [list(p) for p in prompts * 2]
    for _ in range(8):
        added, last = speculative_step(model, cache, last, rows, 3, 3)
        for s, a in zip(seqs, added):
            s += a
    cache.free([0, 4, 2])  # of each prompt one sequence stays
    cache.compact()
    left = [1, 3, 5]
    added, after = speculative_step(model, cache, [last[i] for i in left], cache._ids(left), 3, 3)
    for i, a in zip(left, added):
        seqs[i] += a
    assert cache.status() == 0
    lens, table = cache.seq_lens.tolist(), cache.page_table.long()
    assert [lens[i] for i in left] == [len(seqs[i]) for i in left]
    for i, s in enumerate(seqs):
        n0 = len(prompts[i % 3])
        want, k64, v64 = plain(model, s, torch.float64)
        near, k16, v16 = plain(model, s, dtype)
        margin = 4 * (near.double() - want).abs().max()
        chosen = torch.tensor(s[n0:], device=want.device)
        at = want[n0 - 1:len(s) - 1]
        gap = at.amax(1) - at.gather(1, chosen[:, None])[:, 0]
        assert (gap <= margin).all(), (i, gap.max(), margin)
        assert margin < at.std() / 2  # (a token chosen at random would be far outside)
        if i in left:
            assert want[-1].max() - want[-1, after[left.index(i)]] <= margin
            ids = table[i, :-(-len(s) // 16)]
            for pool, exact, plain16 in ((cache.k, k64, k16), (cache.v, v64, v16)):
                held = pool[:, ids].transpose(2, 3).flatten(1, 2)[:, :len(s)].double()
                off, allowed = (held - exact).abs().amax((1, 2, 3)), (plain16.double() - exact).abs().amax((1, 2, 3))
                assert (off <= 4 * allowed).all(), (i, off, allowed)
                assert (allowed < exact.std() / 4).all()
