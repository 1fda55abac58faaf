"""Speculative decoding over a paged cache, on a small random-init model.

    python examples/speculative_paged.py [--dtype float32] [--steps 24]

Several prompts of different lengths are prefilled as one packed batch
(``prompt_attention``), one of them in two chunks, the second after a prefix in
pages.  Each sequence is then forked for two samples, and every step verifies a
drafted tree per sequence (``tree_attention``), appends the accepted path to the
cache, and in the end the forks give their pages back and the pool is compacted.
Greedy verification must yield the tokens of plain greedy decoding, which the
script checks (in float32, where no two logits tie).
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from adakv_b200.paged import PagedKVCache  # noqa: E402


class TinyLM:
    """Two attention layers with rotary positions and a tied output layer."""

    def __init__(self, vocab=512, width=256, heads=8, kv_heads=2, dim=64, layers=2,
                 dtype=torch.float32, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed)

        def w(*shape, gain=1.0):
            x = torch.randn(shape, generator=g) * gain / shape[-1] ** 0.5
            return x.to(dtype).to(device)

        self.heads, self.kv_heads, self.dim, self.n_layers = heads, kv_heads, dim, layers
        self.embed = w(vocab, width, gain=width ** 0.5)
        self.next = w(width, width, gain=1.0)  # what mostly follows a token: the drafter's guess
        self.wqkv = [w((heads + 2 * kv_heads) * dim, width) for _ in range(layers)]
        self.wo = [w(width, heads * dim, gain=1.0) for _ in range(layers)]

    def rotate(self, x, pos):
        half = self.dim // 2
        f = 10000.0 ** (-torch.arange(half, device=x.device, dtype=torch.float32) / half)
        a = pos[:, None].float() * f
        c, s = a.cos()[:, None], a.sin()[:, None]
        lo, hi = x[..., :half].float(), x[..., half:].float()
        return torch.cat([lo * c - hi * s, hi * c + lo * s], -1).to(x.dtype)

    def forward(self, tokens, pos, attend):
        """Logits of packed tokens and every layer's new k / v ``[layers, T, kv heads,
        dim]``; ``attend(layer, q, k, v)`` is the attention."""
        x = e = self.embed[tokens]
        ks, vs = [], []
        for i in range(self.n_layers):
            h = torch.nn.functional.rms_norm(x, x.shape[-1:])
            q, k, v = (h @ self.wqkv[i].T).unflatten(1, (-1, self.dim)).split(
                [self.heads, self.kv_heads, self.kv_heads], 1)
            q, k = self.rotate(q, pos), self.rotate(k, pos)
            x = x + attend(i, q, k, v).flatten(1) @ self.wo[i].T
            ks.append(k)
            vs.append(v)
        # (without the token's own embedding, whose likeliest next token is itself)
        return (x - e + e @ self.next.T) @ self.embed.T, torch.stack(ks), torch.stack(vs)

    def guesses(self, token, n):
        """The drafter: the n likeliest next tokens by the token alone."""
        return (self.embed[token] @ self.next.T @ self.embed.T).topk(n).indices.tolist()


def prefill(model, cache, prompts, slots):
    """Packed prompts into the rows `slots`; the greedy token after each."""
    dev = cache.k.device
    before = cache.seq_lens[slots.long()].tolist()
    cu = [0]
    for p in prompts:
        cu.append(cu[-1] + len(p))
    tokens = torch.tensor(sum(prompts, []), device=dev)
    pos = torch.cat([torch.arange(len(p)) + b for p, b in zip(prompts, before)]).to(dev)
    cu_t = torch.tensor(cu, dtype=torch.int32, device=dev)
    logits, k, v = model.forward(
        tokens, pos, lambda i, q, k, v: cache.prompt_attention(i, q, k, v, cu_t, slots=slots))
    cache.append(k, v, cu_t, slots=slots)
    return logits[cu_t[1:].long() - 1].argmax(-1).tolist()


def draft(model, token, width, depth):
    """A tree of drafted tokens behind `token` (its own root): tokens, parents, depths."""
    toks, par, dep = [token], [-1], [0]
    level = [0]
    for d in range(1, depth + 1):
        nxt = []
        for node in level:
            for t in model.guesses(toks[node], width):
                nxt.append(len(toks))
                toks.append(t)
                par.append(node)
                dep.append(d)
        level = nxt[:width * 2]  # keep the tree small
    return toks, par, dep


def speculative_step(model, cache, last, slots, width, depth):
    """One step of every row: the tokens that it adds (its last one and the accepted
    ones), and the greedy token after them, which is the next step's first."""
    dev = cache.k.device
    trees = [draft(model, t, width, depth) for t in last]
    cu = [0]
    for t in trees:
        cu.append(cu[-1] + len(t[0]))
    lens = cache.seq_lens[slots.long()].tolist()
    tokens = torch.tensor(sum((t[0] for t in trees), []), device=dev)
    parents = torch.tensor(sum((t[1] for t in trees), []), dtype=torch.int32, device=dev)
    pos = torch.tensor(sum(([d + n for d in t[2]] for t, n in zip(trees, lens)), []), device=dev)
    cu_t = torch.tensor(cu, dtype=torch.int32, device=dev)
    logits, k, v = model.forward(
        tokens, pos, lambda i, q, k, v: cache.tree_attention(i, q, k, v, parents, cu_t, slots=slots))
    best = logits.argmax(-1).tolist()
    paths, after = [], []
    for b, (toks, par, _) in enumerate(trees):
        path = [0]
        while True:
            want = best[cu[b] + path[-1]]
            nxt = [i for i in range(len(toks)) if par[i] == path[-1] and toks[i] == want]
            if not nxt:
                break
            path.append(nxt[0])
        paths.append(path)
        after.append(best[cu[b] + path[-1]])
    w = max(len(p) for p in paths)
    index = torch.tensor([p + [0] * (w - len(p)) for p in paths], dtype=torch.int32, device=dev)
    counts = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=dev)
    cache.append(k, v, cu_t, slots=slots, index=index, counts=counts)
    return [[t[0][i] for i in p] for t, p in zip(trees, paths)], after


def run(dtype=torch.float32, steps=24, width=3, depth=3, seed=0, device="cuda"):
    """Tokens generated per row by trees, the same by single tokens, mean tokens a step."""
    model = TinyLM(dtype=dtype, device=device, seed=seed)
    cache = PagedKVCache(model.n_layers, 400, model.kv_heads, model.dim, 16, n_slots=12,
                         max_seq_len=640, dtype=dtype, device=device)
    g = torch.Generator().manual_seed(seed + 1)
    prompts = [torch.randint(0, 512, (n,), generator=g).tolist() for n in (45, 160, 1)]
    slots = cache._ids([0, 1, 2])
    prefill(model, cache, [prompts[0][:20], prompts[1], prompts[2][:0]], slots)
    last = prefill(model, cache, [prompts[0][20:], [], prompts[2]], slots)
    # (row 1 is whole already: its next token comes from the last prompt token again)
    last[1] = None
    whole = PagedKVCache(model.n_layers, 400, model.kv_heads, model.dim, 16, n_slots=12,
                         max_seq_len=640, dtype=dtype, device=device)
    greedy = prefill(model, whole, prompts, slots)
    last[1] = greedy[1]
    if dtype == torch.float32 and last != greedy:
        raise AssertionError("a prompt in chunks differs from the whole prompt")
    # parallel samples: rows 3 - 5 share the prompts' pages
    cache.fork([0, 1, 2], [3, 4, 5])
    rows = cache._ids([0, 1, 2, 3, 4, 5])
    last = last + last
    out = [[] for _ in range(6)]
    for _ in range(steps):
        added, last = speculative_step(model, cache, last, rows, width, depth)
        for o, a in zip(out, added):
            o += a
    cache.free([3, 4, 5])
    cache.compact()
    more, last3 = speculative_step(model, cache, last[:3], slots, width, depth)  # the pages moved
    for o, a in zip(out, more):
        o += a
    if cache.status():
        raise RuntimeError("a page call failed")
    # plain greedy decoding: trees of one token
    plain, tok = [[] for _ in range(3)], greedy
    for _ in range(max(len(o) for o in out[:3])):
        added, tok = speculative_step(model, whole, tok, slots, 1, 0)
        for o, a in zip(plain, added):
            o += a
    return out, plain, sum(len(o) for o in out) / (6 * steps + 3)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--dtype", default="float32", choices=["float32", "bfloat16", "float16"])
    ap.add_argument("--steps", type=int, default=24)
    a = ap.parse_args()
    out, plain, mean = run(getattr(torch, a.dtype), a.steps)
    same = all(o == p[:len(o)] for o, p in zip(out, plain)) and all(
        out[i + 3] == out[i][:len(out[i + 3])] for i in range(3))
    print(f"{mean:.2f} tokens a step; tokens {'equal' if same else 'differ from'} plain greedy decoding")
    if a.dtype == "float32" and not same:
        raise SystemExit(1)


if __name__ == "__main__":
    main()
