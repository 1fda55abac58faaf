"""Plain 64-bit attention of new tokens, and error bounds from the formula, for
the tests of ``prompt_attention`` and ``tree_attention``."""
import math

import torch

# unit roundoff: half the spacing of numbers with 8, 11 and 24 significant bits
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


class Case:
    """Sequences with `new[b]` new tokens after `prefix[b]` cached ones.  Whatever
    no sequence owns (the rest of a last page, free pages, unused slots, tokens
    outside the sequences) is NaN."""

    def __init__(self, new, prefix, Hq, Hkv, D, dtype, page=16, tree=False, seed=0, gain=1.5,
                 gap=0, device="cuda", shuffle=True):
        g = torch.Generator().manual_seed(seed)
        self.new, self.prefix, self.page, self.dtype = list(new), list(prefix), page, dtype
        self.Hq, self.Hkv, self.D, self.scale = Hq, Hkv, D, 1.0 / math.sqrt(D)
        B = len(self.new)
        self.cu = [gap]
        for n in self.new:
            self.cu.append(self.cu[-1] + n)
        T = self.cu[-1] + gap
        self.T = T

        def rnd(*shape, k=1.0):
            return (torch.randn(shape, generator=g, dtype=torch.float32) * k).to(dtype)

        self.q, self.k, self.v = rnd(T, Hq, D, k=gain), rnd(T, Hkv, D), rnd(T, Hkv, D)
        self.parents = None
        if tree:
            self.parents = torch.full((T,), -1, dtype=torch.int32)
            for b, n in enumerate(self.new):
                for i in range(n):
                    r = int(torch.randint(0, 10, (1,), generator=g))
                    p = max(-1, i - 1 - int(torch.randint(0, 3, (1,), generator=g)))
                    self.parents[self.cu[b] + i] = -2 if r == 0 and i > 0 else p
        owned = torch.zeros(T, dtype=torch.bool)
        owned[self.cu[0]:self.cu[-1]] = True
        if tree:
            owned &= self.parents >= -1
        self.live = owned
        self.k[~owned], self.v[~owned] = math.nan, math.nan
        used = [-(-p // page) for p in self.prefix]
        n_pages = sum(used) + 4
        self.n_slots = B + 2
        self.slots = torch.randperm(self.n_slots, generator=g)[:B] if shuffle else torch.arange(B)
        order = torch.randperm(n_pages, generator=g)
        W = max(max(used, default=0), 1)
        self.table = torch.full((self.n_slots, W), -1, dtype=torch.int32)
        self.lens = torch.zeros(self.n_slots, dtype=torch.int32)
        self.kp = torch.full((n_pages, Hkv, page, D), math.nan, dtype=dtype)
        self.vp = torch.full((n_pages, Hkv, page, D), math.nan, dtype=dtype)
        at = 0
        for b, n in enumerate(used):
            ids = order[at:at + n]
            at += n
            self.table[self.slots[b], :n] = ids.int()
            self.lens[self.slots[b]] = self.prefix[b]
            for j, page_id in enumerate(ids.tolist()):
                m = min(page, self.prefix[b] - j * page)
                self.kp[page_id, :, :m] = rnd(Hkv, m, D)
                self.vp[page_id, :, :m] = rnd(Hkv, m, D)
        self.device = device

    def cu_tensor(self):
        return torch.tensor(self.cu, dtype=torch.int32, device=self.device)

    def pages(self):
        d = self.device
        return self.kp.to(d), self.vp.to(d), self.table.to(d), self.lens.to(d)

    def mask(self, b):
        n, p = self.new[b], self.prefix[b]
        if self.parents is None:
            vis, live = torch.ones(n, n, dtype=torch.bool).tril(), torch.ones(n, dtype=torch.bool)
        else:
            par = self.parents[self.cu[b]:self.cu[b] + n].tolist()
            vis, live = torch.zeros(n, n, dtype=torch.bool), torch.tensor([x >= -1 for x in par], dtype=torch.bool)
            for i in range(n):
                j = i
                while j >= 0 and par[j] >= -1:
                    vis[i, j] = True
                    j = par[j]
        return torch.cat([live[:, None].expand(n, p), vis], 1), live

    def reference(self):
        """out, lse and a bound on the error of each, all float64 (rows that no
        sequence has stay NaN).

        The scores carry at most (D + 4) roundings of 2^-22 (32-bit sums, which
        tensor cores may truncate) of sum |q k| scale; probabilities and their
        sums n + 16 of 2^-22; a 16-bit kernel also rounds each probability once
        to the element type, and the output is rounded once."""
        T, Hq, D = self.T, self.Hq, self.D
        out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
        lse = torch.full((T, Hq), math.nan, dtype=torch.float64)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        u, e = 2.0 ** -22, EPS[self.dtype]
        g = self.Hq // self.Hkv
        for b, n in enumerate(self.new):
            if n == 0:
                continue
            rows = slice(self.cu[b], self.cu[b] + n)
            vis, live = self.mask(b)
            p = self.prefix[b]
            ids = self.table[self.slots[b], :-(-p // self.page)].long()
            for h in range(self.Hkv):
                kc = self.kp[ids, h].reshape(-1, D)[:p]
                vc = self.vp[ids, h].reshape(-1, D)[:p]
                k = torch.cat([kc, torch.where(live[:, None], self.k[rows, h], 0)]).double()
                v = torch.cat([vc, torch.where(live[:, None], self.v[rows, h], 0)]).double()
                for i in range(h * g, h * g + g):
                    q = self.q[rows, i].double()
                    z = torch.where(vis, q @ k.T * self.scale, -math.inf)
                    dz = torch.where(vis, q.abs() @ k.abs().T, 0).amax(1) * self.scale * (D + 4) * u
                    L = torch.logsumexp(z, 1)
                    w = torch.where(live[:, None], torch.exp(z - L[:, None]), 0.0)
                    out[rows, i] = w @ v
                    lse[rows, i] = L
                    a = w @ v.abs()
                    rel = 2 * dz + (n + p + 16) * u + (e if e > u else 0)
                    tol[rows, i] = a * rel[:, None] + out[rows, i].abs() * e + 1e-30
                    if self.dtype == torch.float16:  # the smallest steps of the type
                        tol[rows, i] += 2.0 ** -25
                    ltol[rows, i] = dz + (n + p + 16) * u + L.abs().nan_to_num(0, 0, 0) * u
        return out, lse, tol, ltol

    def check(self, out, lse):
        ref, rl, tol, ltol = self.reference()
        rows = torch.zeros(self.T, dtype=torch.bool)
        rows[self.cu[0]:self.cu[-1]] = True
        o, l = out.double().cpu()[rows], lse.double().cpu()[rows]
        ref, rl, tol, ltol = ref[rows], rl[rows], tol[rows], ltol[rows]
        assert torch.isfinite(o).all()
        bad = (o - ref).abs() > tol
        assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outputs off, worst " \
                              f"{((o - ref).abs() / tol).max():.2f} of the bound"
        dead = rl == -math.inf
        assert (l[dead] == -math.inf).all()
        assert (o[dead.any(1)] == 0).all()
        assert ((l - rl).abs()[~dead] <= ltol[~dead]).all(), \
            f"lse off by {((l - rl).abs() / ltol)[~dead].max():.2f} of the bound"
