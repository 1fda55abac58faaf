"""Cases, inputs and plain forms of the operators over new tokens and paged caches.

Three operators, each over the range it is used in:

``prompt``
    causal attention of packed prompts of different lengths, with grouped
    heads, each after an optional prefix that lies in a paged cache
    (``adakv_b200.prompt.prompt_attention``);
``tree``
    attention of a tree of drafted tokens over a paged cache; one drafted
    token is an ordinary decode step (``adakv_b200.prompt.tree_attention``);
``pages``
    copying pages, forking and freeing sequences, compacting the pool and
    appending tokens (``adakv_b200.paged``).

``run`` computes a case in its plain form (elementary torch operations in 32
bits, rounded once at the end) or, where ``own`` is true, by the framework's
calls.  ``exact`` computes the attention cases in 64 bits, one head at a time.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _ints(text):
    return [int(x) for x in text.split(",")]


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def _attention(name, op, dtype, heads, kv_heads, dim, new, prefix, page=16):
    return {"name": name, "op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "new": new, "prefix": prefix}


def _pages(name, what, dtype, layers, kv_heads, dim, page, pool, seqs, tokens, count):
    return {"name": name, "op": "pages", "what": what, "dtype": dtype, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "pool": pool, "seqs": seqs,
            "tokens": tokens, "count": count}


def listed():
    return [
        # a short chat turn on its own: latency of the smallest prompt
        _attention("prompt_short", "prompt", "bf16", 32, 8, 128, "17", "0"),
        # a server's prefill batch: prompts of one token to 1500, one of them empty
        _attention("prompt_packed", "prompt", "bf16", 32, 8, 128,
                   "1,733,0,1500,64,129,1024,257,90,2", "0,0,0,0,0,0,0,0,0,0"),
        # one long prompt
        _attention("prompt_8k", "prompt", "bf16", 32, 8, 128, "8192", "0"),
        # the next pieces of chunked prompts over what is cached already; groups of 6 heads
        _attention("prompt_chunks", "prompt", "fp16", 12, 2, 64, "512,300,77,1",
                   "4096,1000,0,8191", 32),
        # one token of one long sequence: a plain decode step
        _attention("tree_one_token", "tree", "bf16", 32, 8, 128, "1", "32768"),
        # a server's verification step: 16 sequences of ragged context, trees of 6 to 32 tokens
        _attention("tree_batch", "tree", "bf16", 64, 8, 128,
                   "32,32,16,32,25,32,6,32,32,16,31,32,32,12,32,32",
                   "8191,16384,12000,32768,9001,8192,20000,4097,"
                   "16383,10240,27000,8208,15,6000,12345,30000"),
        # 32-bit verification with odd sizes: groups of 6 heads, pages that end inside a tile
        _attention("tree_fp32", "tree", "fp32", 12, 2, 64, "13,1,64", "1003,0,5000", 32),
        # host-ordered copies of pages (a prefix brought into other pages), 8 layers
        _pages("pages_copy", "copy", "bf16", 8, 8, 128, 16, 2048, 1, 0, 700),
        # eight sequences forked four ways (to 30 new ones) for parallel samples
        _pages("pages_fork", "fork", "bf16", 8, 8, 128, 16, 2048, 40, 800, 30),
        # the pool made dense after sequences have left holes in it
        _pages("pages_compact", "compact", "bf16", 8, 8, 128, 16, 2048, 48, 500, 20),
        # finished sequences leave, some pages of theirs are shared
        _pages("pages_free", "free", "bf16", 1, 8, 128, 16, 16384, 64, 3000, 24),
        # accepted tokens of each verified tree are written behind the cached ones
        _pages("pages_append", "append", "fp16", 8, 8, 128, 32, 1024, 32, 700, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "tree", "tree", "pages"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([16, 32])
    if op == "pages":
        what = rng.choice(["copy", "fork", "compact", "free", "append"])
        layers, kv_heads = _log(rng, 1, 8), rng.choice([1, 2, 4, 8])
        pool = _log(rng, 200, 2048)
        seqs = _log(rng, 4, 40)
        # sequences take at most about half of the pool, so that forks and appends fit
        tokens = max(1, int(pool * page * rng.uniform(0.2, 0.5) / seqs))
        count = _log(rng, 1, pool // 3) if what == "copy" else _log(rng, 1, max(2, seqs // 2))
        if what == "append":
            count = _log(rng, 1, 32)
        case = _pages("", what, dtype, layers, kv_heads, dim, page, pool, seqs, tokens, count)
        del case["name"]
        return case
    kv_heads, group = rng.choice([(8, 4), (8, 8), (2, 6), (1, 16), (4, 1), (6, 5)])
    heads = kv_heads * group
    batch = _log(rng, 1, 24)
    most = 1500 if dtype == "fp32" else 8192
    if op == "prompt":
        new = [_log(rng, 1, most) if rng.random() < 0.95 else 0 for _ in range(batch)]
        prefix = [_log(rng, 1, most) if rng.random() < 0.5 else 0 for _ in range(batch)]
        if rng.random() < 0.5:
            prefix = [0] * batch
        room = 8192 * 8192 * 32 // 2
    else:
        top = _log(rng, 1, 64)
        new = [rng.randint(1, top) for _ in range(batch)]
        prefix = [_log(rng, 16, 4 * most) if rng.random() < 0.95 else 0 for _ in range(batch)]
        room = 16 * 64 * 32 * 32768 // 2
    if dtype == "fp32":
        room //= 8
    if sum(new) == 0:
        new[0] = 1
    # the plain form pads: batch x heads x longest new x longest context scores
    while len(new) > 1 and len(new) * heads * max(new) * (max(prefix) + max(new)) > room:
        new.pop()
        prefix.pop()
    while heads * max(new) * (max(prefix) + max(new)) > room:
        new = [max(1, x * 3 // 4) for x in new]
        prefix = [x * 3 // 4 for x in prefix]
    case = _attention("", op, dtype, heads, kv_heads, dim, ",".join(map(str, new)),
                      ",".join(map(str, prefix)), page)
    del case["name"]
    return case


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _parents(lens, gen):
    """A random tree for each sequence: a token's parent is one of the four tokens
    before it, or (-1) the last cached token; about one in twelve slots of the
    longer trees is unused (-2)."""
    out = []
    for n in lens:
        back = torch.randint(1, 5, (n,), generator=gen)
        at = torch.arange(n)
        p = (at - back).clamp(min=-1)
        dead = (torch.rand(n, generator=gen) < 1 / 12) & (at > 0) & (n > 8)
        # what follows an unused slot hangs off the tree's root instead
        p = torch.where((p >= 0) & dead[p.clamp(min=0)], torch.full_like(p, -1), p)
        out.append(torch.where(dead, torch.full_like(p, -2), p))
    return torch.cat(out).to(torch.int32).to(DEV)


def _prepare_attention(case, gen, cpu_gen):
    dt = TYPES[case["dtype"]]
    new, prefix, ps = _ints(case["new"]), _ints(case["prefix"]), case["page"]
    T, Hq, Hkv, D = sum(new), case["heads"], case["kv_heads"], case["dim"]

    def randn(*shape, gain=1.0):
        return (torch.randn(shape, generator=gen, device=DEV) * gain).to(dt)

    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    used = [-(-p // ps) for p in prefix]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, generator=cpu_gen)[:sum(used)]
    table = torch.full((len(new), max(1, max(used))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    s = {"case": case, "q": randn(T, Hq, D, gain=1.5), "k": randn(T, Hkv, D), "v": randn(T, Hkv, D),
         "cu": _int32(cu), "batch": len(new), "longest": max(new), "longest_prefix": max(prefix),
         "scale": 1.0 / math.sqrt(D), "pages": None}
    if max(prefix) > 0 or case["op"] == "tree":
        s["pages"] = (randn(n_pages, Hkv, ps, D), randn(n_pages, Hkv, ps, D),
                      table.to(DEV), _int32(prefix))
    if case["op"] == "tree":
        s["parents"] = _parents(new, cpu_gen)
    return s


def _prepare_pages(case, gen, cpu_gen):
    dt = TYPES[case["dtype"]]
    L, N, Hkv, ps, D = case["layers"], case["pool"], case["kv_heads"], case["page"], case["dim"]
    B, what = case["seqs"], case["what"]
    shape = (L, N, Hkv, ps, D)
    k = torch.randn(shape, generator=gen, device=DEV, dtype=dt)
    v = torch.randn(shape, generator=gen, device=DEV, dtype=dt)
    s = {"case": case, "k": k, "v": v}
    order = torch.randperm(N, generator=cpu_gen)
    if what == "copy":
        n = min(case["count"], N // 2)
        s["src"], s["dst"] = (order[i * n:(i + 1) * n].to(torch.int32).to(DEV) for i in (0, 1))
        return s
    # sequences of 1 to twice case["tokens"] tokens while the pool has room; three
    # quarters of the slots are empty where forks go there
    held = max(1, B // 4) if what == "fork" else B
    lens, left = [], N * 3 // 4
    if what in ("append", "fork"):
        left = N // 2
    for _ in range(held):
        n = int(torch.randint(1, 2 * case["tokens"] + 1, (1,), generator=cpu_gen))
        n = max(0, min(n, left * ps))
        left -= -(-n // ps)
        lens.append(n)
    lens += [0] * (B - held)
    used = [-(-n // ps) for n in lens]
    width = max(2 * case["tokens"], 1) // ps + 3 + 32 // ps
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    # every fourth sequence shares the full pages of the one before it
    for b in range(3, held, 4):
        n = min(lens[b], lens[b - 1]) // ps
        table[b, :n] = table[b - 1, :n]
    ref = torch.bincount(table[table >= 0].long(), minlength=N).to(torch.int32)
    # one tensor holds the reference counts, the lengths and the page table
    s["meta"] = torch.cat([ref, torch.tensor(lens, dtype=torch.int32), table.reshape(-1)]).to(DEV)
    s["width"] = width
    n = case["count"]
    if what == "fork":
        n = min(n, B - held)
        live = max(1, min(held, -(-n // 4)))
        s["src"] = _int32([i % live for i in range(n)])
        s["dst"] = _int32([held + i for i in range(n)])
    if what == "free":
        s["slots"] = torch.randperm(B, generator=cpu_gen)[:min(n, B)].to(torch.int32).to(DEV)
    if what == "compact":
        # sequences that have left: their pages become holes
        gone = torch.randperm(B, generator=cpu_gen)[:min(n, B - 1)].long()
        rows = table[gone]
        ref -= torch.bincount(rows[rows >= 0].long(), minlength=N).to(torch.int32)
        table[gone] = -1
        for g in gone.tolist():
            lens[g] = 0
        s["meta"] = torch.cat([ref, torch.tensor(lens, dtype=torch.int32), table.reshape(-1)]).to(DEV)
    if what == "append":
        T = B * n
        s["cu"] = _int32([i * n for i in range(B + 1)])
        counts = torch.randint(0, n + 1, (B,), generator=cpu_gen)
        s["counts"] = counts.to(torch.int32).to(DEV)
        # accepted tokens: ascending positions within each sequence's drafted ones
        pick = torch.rand(B, n, generator=cpu_gen).argsort(1)
        pick = torch.where(torch.arange(n)[None] < counts[:, None], pick, torch.full_like(pick, n))
        pick = pick.sort(1).values.clamp(max=n - 1)
        s["index"] = pick.to(torch.int32).to(DEV)
        s["k_new"] = torch.randn((L, T, Hkv, D), generator=gen, device=DEV, dtype=dt)
        s["v_new"] = torch.randn((L, T, Hkv, D), generator=gen, device=DEV, dtype=dt)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cpu_gen = torch.Generator().manual_seed(seed + 1)
    make = _prepare_pages if case["op"] == "pages" else _prepare_attention
    return make(case, gen, cpu_gen)


# --------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------
def _padded(s):
    """Each sequence's positions in a [batch, longest] grid: indices of the packed
    tokens and which of them exist."""
    cu = s["cu"].long()
    lens = cu[1:] - cu[:-1]
    at = torch.arange(s["longest"], device=DEV)
    return (cu[:-1, None] + at).clamp(max=max(0, s["q"].shape[0] - 1)), at < lens[:, None]


def _plain_attention(s):
    case, B = s["case"], s["batch"]
    Hq, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    where, there = _padded(s)
    n = s["longest"]
    at = torch.arange(n, device=DEV)
    if case["op"] == "tree":
        par = torch.where(there, s["parents"][where].long(), torch.full_like(where, -2))
        live = par >= -1
        seen = torch.eye(n, device=DEV, dtype=torch.bool) | (par[:, :, None] == at)
        steps = max(1, (n - 1).bit_length())
        for _ in range(steps):  # ancestors at up to 2, 4, 8 ... links
            seen = (seen.float() @ seen.float()) > 0
        seen = seen & live[:, :, None] & live[:, None, :]
    else:
        live = there
        seen = (at[:, None] >= at[None]) & there[:, :, None] & there[:, None, :]
    q = s["q"][where].float().reshape(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    k = torch.where(there[..., None, None], s["k"][where].float(), 0.0).permute(0, 2, 1, 3)
    v = torch.where(there[..., None, None], s["v"][where].float(), 0.0).permute(0, 2, 1, 3)
    if s["pages"] is not None and s["longest_prefix"] > 0:
        kp, vp, table, lens = s["pages"]
        ps, m = case["page"], s["longest_prefix"]
        old = torch.arange(m, device=DEV)
        held = old < lens[:, None]
        page = table[:, old // ps].long().clamp(min=0)
        kc = torch.where(held[..., None, None], kp[page, :, old % ps].float(), 0.0)
        vc = torch.where(held[..., None, None], vp[page, :, old % ps].float(), 0.0)
        k = torch.cat([kc.permute(0, 2, 1, 3), k], 2)
        v = torch.cat([vc.permute(0, 2, 1, 3), v], 2)
        seen = torch.cat([held[:, None, :] & live[:, :, None], seen], 2)
    z = (q @ k[:, :, None].transpose(-1, -2)) * s["scale"]
    z.masked_fill_(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = z.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    out = (e @ v[:, :, None]) / torch.where(total == 0, 1.0, total)
    lse = (total.log() + top)[..., 0]
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[there].to(s["q"].dtype)
    return {"out": out, "lse": lse.permute(0, 3, 1, 2).reshape(B, n, Hq)[there]}


def _split_meta(s):
    N, B = s["case"]["pool"], s["case"]["seqs"]
    meta = s["meta"].clone()  # every pass starts from the same sequences
    return meta[:N], meta[N:N + B], meta[N + B:].view(B, s["width"])


def _plain_pages(s):
    case, k, v = s["case"], s["k"], s["v"]
    what, ps = case["what"], case["page"]
    if what == "copy":
        src, dst = s["src"].long(), s["dst"].long()
        k[:, dst] = k[:, src]
        v[:, dst] = v[:, src]
        return {"k": k, "v": v}
    ref, lens, table = _split_meta(s)
    cols = torch.arange(table.shape[1], device=DEV)
    if what == "free":
        rows = table[s["slots"].long()]
        gone = rows[rows >= 0].long()
        ref.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
        table[s["slots"].long()] = -1
        lens[s["slots"].long()] = 0
        return {"ref": ref, "lens": lens, "table": table}
    if what == "fork":
        src, dst = s["src"].long(), s["dst"].long()
        n = lens[src]
        full, part = n // ps, n % ps > 0
        free = torch.nonzero(ref == 0)[:, 0].to(torch.int32)
        fresh = free[(part.cumsum(0) - 1).clamp(min=0)]
        rows = table[src]
        shared = rows[cols < full[:, None]].long()
        tail = torch.gather(rows, 1, full[:, None].long())[:, 0]
        rows = torch.where((cols == full[:, None]) & part[:, None], fresh[:, None], rows)
        table[dst] = rows
        lens[dst] = n
        ref.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
        to, by = fresh[part].long(), tail[part].long()
        ref[to] = 1
        k[:, to] = k[:, by]
        v[:, to] = v[:, by]
    if what == "compact":
        live = ref > 0
        count = live.sum()
        ids = torch.arange(ref.shape[0], device=DEV)
        moved = ids[live & (ids >= count)]
        holes = ids[~live & (ids < count)]
        new = ids.to(torch.int32)
        new[moved] = holes.to(torch.int32)
        table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()], table))
        ref[holes] = ref[moved]
        ref[moved] = 0
        k[:, holes] = k[:, moved]
        v[:, holes] = v[:, moved]
    if what == "append":
        n = s["counts"]
        after = lens + n
        have, need = (lens + ps - 1) // ps, (after + ps - 1) // ps
        free = torch.nonzero(ref == 0)[:, 0].to(torch.int32)
        takes = need - have
        first = takes.cumsum(0) - takes
        mine = (cols >= have[:, None]) & (cols < need[:, None])
        fresh = free[(first[:, None] + cols - have[:, None]).clamp(0, free.shape[0] - 1)]
        table.copy_(torch.where(mine, fresh, table))
        ref[table[mine].long()] = 1
        i = torch.arange(s["index"].shape[1], device=DEV)
        kept = i < n[:, None]
        to = lens[:, None] + i
        page = torch.gather(table, 1, (to // ps).clamp(max=table.shape[1] - 1).long())[kept].long()
        place = (to % ps)[kept].long()
        by = (s["cu"][:-1, None] + s["index"])[kept].long()
        # the two indexed axes are apart, so they come first: [accepted, layer, head, dim]
        k[:, page, :, place] = s["k_new"][:, by].transpose(0, 1)
        v[:, page, :, place] = s["v_new"][:, by].transpose(0, 1)
        lens.copy_(after)
    return {"k": k, "v": v, "ref": ref, "lens": lens, "table": table}


# --------------------------------------------------------------------------
# the framework's calls
# --------------------------------------------------------------------------
def _own_attention(s):
    from adakv_b200.prompt import prompt_attention, tree_attention
    if s["case"]["op"] == "tree":
        out, lse = tree_attention(s["q"], s["k"], s["v"], s["parents"], s["cu"], *s["pages"],
                                  scale=s["scale"], return_lse=True)
    else:
        out, lse = prompt_attention(s["q"], s["k"], s["v"], s["cu"], prefix=s["pages"],
                                    scale=s["scale"], return_lse=True)
    return {"out": out, "lse": lse}


def _own_pages(s):
    from adakv_b200 import paged
    k, v, what = s["k"], s["v"], s["case"]["what"]
    if what == "copy":
        paged.copy_pages(k, v, s["src"], s["dst"])
        return {"k": k, "v": v}
    ref, lens, table = _split_meta(s)
    if what == "free":
        paged.free_sequences(table, lens, ref, s["slots"])
        return {"ref": ref, "lens": lens, "table": table}
    if what == "fork":
        paged.fork_sequences(k, v, table, lens, ref, s["src"], s["dst"])
    if what == "compact":
        paged.compact_pages(k, v, table, lens, ref)
    if what == "append":
        paged.append_tokens(k, v, table, lens, ref, s["k_new"], s["v_new"], s["cu"],
                            index=s["index"], counts=s["counts"])
    return {"k": k, "v": v, "ref": ref, "lens": lens, "table": table}


def run(s):
    if s["case"]["op"] == "pages":
        return _own_pages(s) if own else _plain_pages(s)
    return _own_attention(s) if own else _plain_attention(s)


# --------------------------------------------------------------------------
# the least work, and the result in 64 bits
# --------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    D, Hkv = case["dim"], case["kv_heads"]
    if case["op"] != "pages":
        new, prefix, Hq = _ints(case["new"]), _ints(case["prefix"]), case["heads"]
        T = sum(new)
        # the drafted tokens' own pairs: their causal triangle (a chain's, the most a tree has)
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, prefix))
        kept = sum(p for n, p in zip(new, prefix) if n)
        return {"bytes": size * D * (2 * T * Hq + 2 * Hkv * (T + kept)) + 4 * T * Hq,
                "flops": 4 * D * Hq * pairs}
    page = 2 * case["layers"] * Hkv * case["page"] * D * size
    N, B = case["pool"], case["seqs"]
    if case["what"] == "copy":
        return {"bytes": 2 * page * min(case["count"], N // 2), "flops": 0}
    rows = case["tokens"] // case["page"] + 1  # a mean sequence's pages
    n = min(case["count"], B)
    if case["what"] == "free":
        return {"bytes": 4 * (4 * n * rows + 2 * n), "flops": 0}
    if case["what"] == "fork":
        n = min(n, B - max(1, B // 4))
        return {"bytes": 2 * page * n + 4 * (4 * n * rows), "flops": 0}
    if case["what"] == "compact":
        # holes below the live count: about a quarter of what is live moves
        live = max(1, min(N * 3 // 4, (B - n) * rows))
        return {"bytes": 2 * page * max(1, live // 4) + 4 * (2 * N + 2 * B * rows), "flops": 0}
    return {"bytes": 2 * page * B * case["count"] // (2 * case["page"]) + 4 * N, "flops": 0}


def exact(case, seed):
    if case["op"] == "pages":
        return None  # moves values, computes none
    s = prepare(case, seed)
    new, prefix, ps = _ints(case["new"]), _ints(case["prefix"]), case["page"]
    Hq, Hkv = case["heads"], case["kv_heads"]
    if sum(n * (n + p) for n, p in zip(new, prefix)) * Hq * case["dim"] > 1e13:
        return None
    T = sum(new)
    out = torch.zeros(T, Hq, case["dim"], dtype=torch.float64, device=DEV)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=DEV)
    begin = 0
    for b, (n, p) in enumerate(zip(new, prefix)):
        if n == 0:
            continue
        rows = slice(begin, begin + n)
        begin += n
        if case["op"] == "tree":
            par = s["parents"][rows].tolist()
            vis = torch.zeros(n, n, dtype=torch.bool)
            for i in range(n):
                j = i if par[i] >= -1 else -1
                while j >= 0:
                    vis[i, j] = True
                    j = par[j]
            live = torch.tensor([x >= -1 for x in par])
        else:
            vis = torch.ones(n, n, dtype=torch.bool).tril()
            live = torch.ones(n, dtype=torch.bool)
        vis = torch.cat([live[:, None].expand(n, p), vis], 1).to(DEV)
        for h in range(Hkv):
            k, v = s["k"][rows, h].double(), s["v"][rows, h].double()
            if p:
                pages = s["pages"][2][b, :-(-p // ps)].long()
                k = torch.cat([s["pages"][0][pages, h].reshape(-1, case["dim"])[:p].double(), k])
                v = torch.cat([s["pages"][1][pages, h].reshape(-1, case["dim"])[:p].double(), v])
            for i in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                z = s["q"][rows, i].double() @ k.T * s["scale"]
                z = torch.where(vis, z, -math.inf)
                lse[rows, i] = torch.logsumexp(z, 1)
                w = torch.where(live.to(DEV)[:, None], torch.softmax(z, 1), 0.0)
                out[rows, i] = w @ v
    return {"out": out, "lse": lse}
