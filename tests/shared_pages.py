"""Steps over a page pool that streams share, and what the ops over it give, in 64 bits straight from the definitions."""
import math

import torch


class Step:
    """`groups`: list of (shared tokens, [own stream, ..]); `alone`: streams of no group. A stream is a list of its rows' context lengths (a length counts the
    shared tokens). Pages lie in no order; whatever no row sees is `poison`, in keys and values."""

    def __init__(self, g, dev, nq, nkv, hd, page, groups=(), alone=(), dtype=torch.bfloat16, poison=float("nan"), spare=3, width=0, gap=0, q_scale=1.0):
        self.nq, self.nkv, self.hd, self.page = nq, nkv, hd, page
        streams, self.member = [], []
        for gi, (shared, members) in enumerate(groups):
            for m in members:
                streams.append(list(m))
                self.member.append(gi)
        for m in alone:
            streams.append(list(m))
            self.member.append(None)
        self.streams, self.shared = streams, [s for s, _ in groups]
        pages_for = lambda n: (n + page - 1) // page
        S = len(streams)
        longest = [max(list(r) + [0]) for r in streams]
        first = {gi: self.member.index(gi) for gi in range(len(groups)) if gi in self.member}
        need = [pages_for(max(longest[s], self.shared[self.member[s]] if first.get(self.member[s]) == s else 0)) for s in range(S)]
        per = max(need + [1]) + width
        total = sum(need) + spare
        order = torch.randperm(total, generator=g, device=dev).int()
        self.table, at = torch.full((S + gap, per), -1, dtype=torch.int32, device=dev), 0
        self.slots = [s + gap for s in range(S)]
        for s in range(S):
            have = 0
            if self.member[s] is not None and first[self.member[s]] != s:
                # whole shared pages are the first stream's; a page that the shared tokens end in is the stream's own, its first tokens are not read
                have = min(self.shared[self.member[s]] // page, need[s])
                self.table[s + gap, :have] = self.table[first[self.member[s]] + gap, :have]
            self.table[s + gap, have:need[s]] = order[at:at + need[s] - have]
            at += need[s] - have
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
        counts = [len(r) for r in streams]
        row0 = [sum(counts[:s]) for s in range(S)]
        self.rows = sum(counts)
        self.kvlen = i32([n for r in streams for n in r])
        self.segs = (i32(self.slots), i32(row0), i32(counts), max(counts + [0]))
        self.groups = None
        if groups:
            self.groups = (i32([first[gi] for gi in range(len(groups))]), i32([len(m) for _, m in groups]), i32(self.shared))
        self.row_seg = [s for s, r in enumerate(streams) for _ in r]
        self.first = first
        rnd = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.q = (rnd(self.rows, nq, hd) * q_scale).to(dtype)
        self.k, self.v = rnd(total, page, nkv, hd).to(dtype), rnd(total, page, nkv, hd).to(dtype)
        if poison is not None:
            seen = torch.zeros(total * page, dtype=torch.bool, device=dev)
            for t in range(self.rows):
                seen[self.at(t)] = True
            self.k.view(-1, nkv, hd)[~seen] = poison
            self.v.view(-1, nkv, hd)[~seen] = poison
        self.mass = torch.rand(total, nkv, page, generator=g, device=dev) * 3

    def at(self, t):
        """Cache rows of the tokens that row t sees."""
        s = self.row_seg[t]
        n = int(self.kvlen[t])
        pos = torch.arange(max(n, 0), device=self.table.device)
        own = self.table[self.slots[s]]
        if self.member[s] is None:
            page = own[pos // self.page]
        else:
            gi = self.member[s]
            page = torch.where(pos < self.shared[gi], self.table[self.slots[self.first[gi]]][pos // self.page], own[pos // self.page])
        return page.long() * self.page + pos % self.page

    def args(self):
        return self.table, self.page, self.nq, self.nkv, self.hd

    def weights(self, t):
        """Scores, logarithm of their sum, weights of row t: [nkv, share, tokens], and what rounding of 32-bit sums leaves of a score."""
        k = self.k.reshape(-1, self.nkv, self.hd)[self.at(t)].double()
        q = self.q[t].reshape(self.nkv, -1, self.hd).double()
        x = torch.einsum("kgd,tkd->kgt", q, k) / math.sqrt(self.hd)
        l = torch.logsumexp(x, -1)
        # a sum of hd products in 32 bits: off by 2^-20 of the sum of their magnitudes at most (hd / 16 steps of the tensor cores, 2^-22 each)
        off = (torch.einsum("kgd,tkd->kgt", q.abs(), k.abs()) / math.sqrt(self.hd)).amax(-1) * 2.0 ** -20 if k.shape[0] else torch.zeros_like(l)
        return x, l, off

    def attend(self):
        """out [rows, nq, hd], lse [rows, nq] and how far each may be off in 32-bit arithmetic with weights of twice eight bits, before out is rounded."""
        dev = self.q.device
        out = torch.zeros(self.rows, self.nq, self.hd, dtype=torch.float64, device=dev)
        lse = torch.full((self.rows, self.nq), -math.inf, dtype=torch.float64, device=dev)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        for t in range(self.rows):
            if int(self.kvlen[t]) <= 0:
                continue
            x, l, off = self.weights(t)
            p = torch.exp(x - l[..., None])
            v = self.v.reshape(-1, self.nkv, self.hd)[self.at(t)].double()
            out[t] = torch.einsum("kgt,tkd->kgd", p, v).reshape(self.nq, self.hd)
            lse[t] = l.reshape(-1)
            # a weight: its score's error and 2^-21 of the exponential, once above and once below the fraction; above it the weight is a bf16 number and what that
            # leaves, at most 2^-8 of it, another one: off by 2^-16 of it. Its product is added in fewer than 2^10 steps (eight for 64 keys), 2^-22 each.
            tol[t] = (torch.einsum("kgt,tkd->kgd", p, v.abs()) * (2 * (off[..., None] + 2.0 ** -20) + 2.0 ** -16 + 2.0 ** -12)).reshape(self.nq, self.hd)
            ltol[t] = (off + 2.0 ** -22 * l.abs() + 2.0 ** -20).reshape(-1)
        return out, lse, tol, ltol

    def spans(self):
        """Cache rows whose sums a step touches."""
        seen = torch.zeros(self.k.shape[0] * self.page, dtype=torch.bool, device=self.q.device)
        for t in range(self.rows):
            seen[self.at(t)] = True
        return seen

    def masses(self, carry, lse=None, start=None):
        """New sums [pages, nkv, page] (entries that no key of the step has stay as in `start`) and how far they may be off."""
        mass = self.mass if start is None else start
        new = torch.zeros(self.k.shape[0] * self.page, self.nkv, dtype=torch.float64, device=self.q.device)
        tol = torch.zeros_like(new)
        for t in range(self.rows):
            if int(self.kvlen[t]) <= 0:
                continue
            x, l, off = self.weights(t)
            ll = l if lse is None else lse[t].reshape(self.nkv, -1).double()
            p = torch.exp(x - ll[..., None])
            rel = off[..., None] * 2 + 2.0 ** -20 + 2.0 ** -22 * (x.abs() + ll[..., None].abs())
            at = self.at(t)
            new.index_add_(0, at, p.sum(1).t())
            tol.index_add_(0, at, (p * rel).sum(1).t())
        tol += new * (self.rows * self.nq // self.nkv) * 2.0 ** -24
        shape = lambda y: y.view(-1, self.page, self.nkv).transpose(1, 2)
        seen = self.spans().view(-1, 1, self.page)
        base = mass.double() * carry if carry else torch.zeros_like(mass, dtype=torch.float64)
        want = torch.where(seen, shape(new) + base, mass.double())
        return want, torch.where(seen, shape(tol) + 2.0 ** -22 * (base.abs() + shape(new)), torch.zeros_like(want)), seen.expand_as(want)


def evicted(mass, n, keep, first, recent):
    """Tokens that stay of n with these sums: [..] python numbers, straight from the definition."""
    if n <= keep:
        return list(range(n))
    middle = sorted(range(first, n - recent), key=lambda i: (0 if math.isnan(mass[i]) else 1, -mass[i] if not math.isnan(mass[i]) else 0.0, i))
    return sorted(list(range(first)) + middle[:keep - first - recent] + list(range(n - recent, n)))
