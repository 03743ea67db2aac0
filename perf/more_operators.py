"""What serving does with a page pool that streams share, as calls that can be timed and checked: attention of a batch whose streams have a long
prefix in common, the weight that a step's queries gave to every cached key, and the move of the heaviest keys into fewer pages.

Caches are [pages, page, kv heads, dim]; the pages of a stream are a row of `table`. Streams of a group hold the same pages at the head of their rows,
`shared` tokens (whole pages); behind them every stream has pages of its own. A step has `rows` rows a stream, its last tokens; row i sees the first
`row_kvlen[i]` tokens of its stream.

* attend: o = softmax(q . k / sqrt(dim)) v over what the row sees, and the logarithm of the softmax's sum (natural, of the scaled scores).
* mass: per kv head and key, the sum of these weights over the step's rows and the heads that share the kv head, added to `carry` times the sum so
  far. Sums are [pages, kv heads, page] in 32 bits, beside the cache's pages. Decoding steps have the logarithms of their attention in hand, prompts do not.
* evict: per stream and kv head, the `first` first tokens, the `recent` last ones and of the others the heaviest, `keep` in all (the earliest of
  equal ones), move in their order to new pages: keys, values, their scales where the cache has codes of 8 bits, and sums.
"""
from __future__ import annotations

import math

import torch

own = False

SPARE = 1.1                  # pages in a pool beyond those in use


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    """`groups` of `streams` streams with `shared` tokens in common, `alone` streams beside them, `own` tokens more in the longest; `rows` new tokens per
    stream. `heads` query heads, `kv` of keys and values, `dim` wide; `page` tokens a page."""
    attend = lambda name, streams, shared, own, heads, kv, dim, rows=1, groups=1, alone=0, page=64: dict(
        name=name, do="attend", groups=groups, streams=streams, alone=alone, shared=shared, own=own, heads=heads, kv=kv, dim=dim, rows=rows, page=page)
    mass = lambda name, streams, shared, own, heads, kv, dim, rows=1, groups=1, alone=0, page=64: dict(
        attend(name, streams, shared, own, heads, kv, dim, rows, groups, alone, page), do="mass")
    evict = lambda name, streams, own, keep, first, recent, kv, dim, bits=16, page=64: dict(
        name=name, do="evict", groups=0, streams=0, alone=streams, shared=0, own=own, keep=keep, first=first, recent=recent, heads=kv, kv=kv, dim=dim,
        bits=bits, rows=1, page=page)
    return [
        # two answers to one prompt: latency
        attend("attend-2", 2, 1024, 100, 24, 4, 256),
        # a few users of one assistant, whose instructions they share
        attend("attend-6", 6, 8000, 900, 24, 4, 256),
        # many agents over one document, and two streams of something else
        attend("attend-32", 32, 30000, 2000, 24, 4, 256, alone=2),
        # many samples of one very long prompt
        attend("attend-64", 64, 60000, 500, 32, 8, 128),
        # drafted tokens of two groups verified on a model with few kv heads
        attend("attend-verify", 4, 5003, 700, 16, 2, 256, rows=9, groups=2),
        # a decode step of a few users of one assistant
        mass("mass-6", 6, 8000, 900, 24, 4, 256),
        # one stream far into a long document
        mass("mass-1-long", 0, 0, 100000, 24, 4, 256, groups=0, alone=1),
        # a chunk of a long prompt
        mass("mass-prompt", 0, 0, 16000, 24, 4, 256, rows=2048, groups=0, alone=1),
        # a prompt's odd end on narrower heads
        mass("mass-prompt-1111", 0, 0, 5000, 32, 8, 128, rows=1111, groups=0, alone=1),
        # a stream that has outgrown its share of the pool
        evict("evict-1", 1, 4000, 1024, 4, 256, 4, 256),
        # all streams of a loaded server
        evict("evict-24", 24, 12000, 2048, 4, 512, 4, 256),
        # two very long ones in a cache of 8 bits
        evict("evict-fp8", 2, 100000, 8192, 16, 1000, 2, 256, bits=8),
    ]


HEADS = [(24, 4, 256), (16, 2, 256), (32, 8, 128), (20, 4, 128), (6, 6, 128), (4, 2, 64), (24, 3, 64)]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    do, page = rng.choice(["attend", "attend", "mass", "mass", "evict"]), rng.choice([64, 64, 128])
    heads, kv, dim = rng.choice(HEADS)
    case = dict(do=do, heads=heads, kv=kv, dim=dim, page=page, groups=0, streams=0, alone=0, shared=0, rows=1)
    room = 60000 * 8 * 128 // (kv * dim)                                 # tokens whose keys and values are as many bytes as the largest case's
    if do == "evict":
        case["alone"], case["bits"] = log(1, 32), rng.choice([16, 16, 8])
        case["own"] = log(1, min(100000, 24 * 12000 * 4 // (kv * case["alone"])))
        case["keep"] = min(log(1, 8192), 24 * 2048 * 1024 // (kv * dim * case["alone"]) + 1)
        case["first"] = rng.choice([0, min(case["keep"] // 4, 4)])
        case["recent"] = rng.randint(0, case["keep"] - case["first"])
        case["heads"] = kv
        return case
    kind = rng.choice(["decode", "decode", "verify"] if do == "attend" else ["decode", "verify", "prompt"])
    if kind == "prompt":
        case["alone"] = rng.choice([1, 1, 2, 3])
        case["rows"] = max(1, log(33, 2048) // case["alone"])
        case["own"] = max(case["rows"], log(40, min(16000, 16000 * 24 * 256 // (heads * dim))))
        return case
    case["rows"] = 1 if kind == "decode" else log(2, 17)
    case["groups"] = rng.choice([0, 1, 1, 1, 2, 3])
    most = 64 // case["rows"]
    case["streams"] = log(2, max(2, most // max(1, case["groups"]))) if case["groups"] else 0
    case["alone"] = rng.choice([0, 1, 3]) if case["groups"] else log(1, max(1, most))
    n = case["groups"] * case["streams"] + case["alone"]
    case["own"] = max(case["rows"], log(1, max(2, room // (2 * n))))
    while case["groups"]:
        case["shared"] = log(page, max(2 * page, room // (2 * case["groups"])))
        if case["shared"] * heads * dim * n * case["rows"] <= 60000 * 32 * 128 * 64:
            break
    return case


def contexts(case):
    """(group or None, tokens) of every stream: its shared pages and its own tokens, unequal ones."""
    shared = case["shared"] // case["page"] * case["page"]               # whole pages; what is left of the shared text is every stream's own
    left = case["shared"] - shared
    out, n = [], case["groups"] * case["streams"] + case["alone"]
    for i in range(n):
        mine = max(case["rows"], int(case["own"] * (1 - 0.7 * ((i * 0.618) % 1))))
        g = i // case["streams"] if i < case["groups"] * case["streams"] else None
        out.append((g, shared + left + mine if g is not None else mine))
    return out


def shared_tokens(case):
    return case["shared"] // case["page"] * case["page"]


# ---- inputs ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    """What the engine has in hand: the page pool with every stream's context in it, the step's tables and queries. Queries and keys as they come out of
    a norm over the head; one token in 64 lies in a direction that a head's queries share (what a real model attends to heavily)."""
    g = torch.Generator("cuda").manual_seed(seed * 7919 + 23)
    dev, page, kv, dim, heads, rows = "cuda", case["page"], case["kv"], case["dim"], case["heads"], case["rows"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    ctx, whole = contexts(case), shared_tokens(case) // page
    per = max((n + page - 1) // page for _, n in ctx)
    used = sum((n + page - 1) // page for _, n in ctx)
    keep_pages = len(ctx) * ((case["keep"] + page - 1) // page) if case["do"] == "evict" else 0
    n_src = int(used * SPARE) + 1
    order = torch.randperm(n_src, generator=g, device=dev).int()
    table, at, held = torch.full((len(ctx), per), -1, dtype=torch.int32, device=dev), 0, {}
    for s, (grp, n) in enumerate(ctx):
        k, have = (n + page - 1) // page, 0
        if grp is not None:
            if grp not in held:
                held[grp] = order[at:at + whole]
                at += whole
            table[s, :whole] = held[grp]
            have = whole
        table[s, have:k] = order[at:at + k - have]
        at += k - have
    S = len(ctx)
    st = dict(case=case, table=table, ctx=ctx)
    st["seg_slot"], st["seg_row0"], st["seg_nrows"] = i32(list(range(S))), i32([s * rows for s in range(S)]), i32([rows] * S)
    st["row_kvlen"] = i32([n - rows + r + 1 for _, n in ctx for r in range(rows)])
    st["grp_seg0"] = i32([j * case["streams"] for j in range(case["groups"])])
    st["grp_nsegs"] = i32([case["streams"]] * case["groups"])
    st["grp_len"] = i32([shared_tokens(case)] * case["groups"])
    toks = (n_src + keep_pages) * page
    way = torch.randn(kv, dim, generator=g, device=dev)                  # the direction
    k = torch.empty(toks, kv, dim, dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    for lo in range(0, toks, 1 << 14):
        n = min(1 << 14, toks - lo)
        loud = (torch.rand(n, kv, 1, generator=g, device=dev) < 1 / 64).float() * torch.rand(n, kv, 1, generator=g, device=dev)
        k[lo:lo + n] = torch.randn(n, kv, dim, generator=g, device=dev) + loud * way * (12 / dim ** 0.5)
        v[lo:lo + n] = torch.randn(n, kv, dim, generator=g, device=dev)
    if case["do"] == "evict":
        move = lambda x: x.view(-1, page, *x.shape[1:])
        st["seg_len"] = i32([n for _, n in ctx])
        st["dst"] = torch.randperm(keep_pages, generator=g, device=dev).int().view(S, -1) + n_src
        st["first_dst"] = n_src
        k[n_src * page:] = 0
        v[n_src * page:] = 0
        mass = torch.randn(n_src + keep_pages, kv, page, generator=g, device=dev).mul_(2).exp_()
        mass[torch.rand(mass.shape, generator=g, device=dev) < 0.1] = 0              # keys that no query has looked at
        mass[n_src:] = 0
        st["mass"] = mass
        st["scale"] = None
        if case["bits"] == 8:
            st["scale"] = torch.rand(toks, kv, 2, generator=g, device=dev).add_(0.5).div_(64)
            st["scale"][n_src * page:] = 0
            k, v = ((x.float() * 32).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for x in (k, v))
            st["scale"] = move(st["scale"])
        st["k"], st["v"] = move(k), move(v)
    else:
        T = S * rows
        q = torch.randn(T, heads, dim, generator=g, device=dev)
        q = q + way.repeat_interleave(heads // kv, 0) * (torch.rand(T, heads, 1, generator=g, device=dev) * 6 / dim ** 0.5)
        st["q"] = q.to(torch.bfloat16)
        st["k"], st["v"] = k.view(-1, page, kv, dim), v.view(-1, page, kv, dim)
        if case["do"] == "mass":
            st["mass"] = torch.rand(n_src, kv, page, generator=g, device=dev) * 4
            st["out"] = st["mass"].clone()
            st["lse"] = None
            if rows <= 32:                                               # the step's attention has left them behind
                st["lse"] = torch.empty(T, heads, device=dev)
                for s in range(S):
                    for h in range(kv):
                        sc = scores(st, s, h)
                        top = sc.amax(-1, keepdim=True)
                        st["lse"].view(T, kv, -1)[s * rows:(s + 1) * rows, h] = ((sc - top).exp().sum(-1, keepdim=True).log() + top)[..., 0]
    if own:
        from ferrite_b200.ops.cuda_ops import CudaOps
        st["ops"] = CudaOps(dev)
    return st


def token_rows(st, s, n):
    """Numbers of the cache rows of the first n tokens of stream s."""
    page = st["case"]["page"]
    pos = torch.arange(n, device=st["table"].device)
    return st["table"][s, pos // page].long() * page + pos % page


def scores(st, s, h):
    """Scaled scores of stream s's rows, heads of kv head h: [rows, heads / kv, tokens] in 32 bits, -inf where a row does not see the key."""
    case, n = st["case"], st["ctx"][s][1]
    rows, kv, dim = case["rows"], case["kv"], case["dim"]
    keys = st["k"].view(-1, kv, dim)[token_rows(st, s, n), h].float()
    q = st["q"].view(-1, kv, case["heads"] // kv, dim)[s * rows:(s + 1) * rows, h].float()
    sc = (q @ keys.t()) / math.sqrt(dim)
    sees = torch.arange(n, device=keys.device)[None, None] < st["row_kvlen"][s * rows:(s + 1) * rows, None, None]
    return torch.where(sees, sc, torch.full_like(sc, float("-inf")))


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(st):
    return run_own(st) if own else run_plain(st)


def run_own(st):
    case, ops = st["case"], st["ops"]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    if case["do"] == "evict":
        kept = ops.kv_evict(st["k"], st["v"], st["scale"], st["mass"], st["seg_slot"], st["seg_len"], st["table"], st["dst"], page, case["keep"],
                            case["first"], case["recent"])
        return moved(st, kept)
    segs = (st["seg_slot"], st["seg_row0"], st["seg_nrows"], case["rows"])
    groups = (st["grp_seg0"], st["grp_nsegs"], st["grp_len"]) if case["groups"] else None
    if case["do"] == "attend":
        return ops.attention_shared(st["q"], None, st["k"], st["v"], st["row_kvlen"], st["table"], page, heads, kv, dim, False, segs, groups, want_lse=True)
    return ops.attention_mass(st["q"], st["k"], st["mass"], st["row_kvlen"], st["table"], page, heads, kv, dim, segs, groups, lse=st["lse"], carry=0.75,
                              out=st["out"])


def moved(st, kept):
    """The tokens kept and the new pages (codes of 8 bits as the numbers that they stand for beside their scales)."""
    at = st["first_dst"]
    k, v = st["k"][at:], st["v"][at:]
    if st["scale"] is None:
        return kept, k, v, st["mass"][at:]
    return kept, k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), st["scale"][at:], st["mass"][at:]


def run_plain(st):
    case = st["case"]
    heads, kv, dim, page, rows = case["heads"], case["kv"], case["dim"], case["page"], case["rows"]
    if case["do"] == "attend":
        out = torch.empty(len(st["ctx"]) * rows, kv, heads // kv, dim, dtype=torch.bfloat16, device="cuda")
        lse = torch.empty(out.shape[:3], device="cuda")
        for s, (_, n) in enumerate(st["ctx"]):
            at = token_rows(st, s, n)
            for h in range(kv):
                sc = scores(st, s, h)
                top = sc.amax(-1, keepdim=True)
                p = (sc - top).exp()
                total = p.sum(-1, keepdim=True)
                out[s * rows:(s + 1) * rows, h] = ((p / total) @ st["v"].view(-1, kv, dim)[at, h].float()).to(torch.bfloat16)
                lse[s * rows:(s + 1) * rows, h] = (total.log() + top)[..., 0]
        return out.view(-1, heads * dim), lse.view(-1, heads)
    if case["do"] == "mass":
        sums = torch.zeros(st["mass"].shape[0] * page, kv, dtype=torch.float64, device="cuda")       # long sums
        seen = torch.zeros(sums.shape[0], dtype=torch.bool, device="cuda")
        for s, (_, n) in enumerate(st["ctx"]):
            at = token_rows(st, s, n)
            seen[at] = True
            for h in range(kv):
                sc = scores(st, s, h)
                if st["lse"] is None:
                    p = (sc - sc.amax(-1, keepdim=True)).exp()
                    p = p / p.sum(-1, keepdim=True)
                else:
                    p = (sc - st["lse"].view(-1, kv, heads // kv)[s * rows:(s + 1) * rows, h, :, None]).exp()
                sums[:, h].index_add_(0, at, p.sum((0, 1), dtype=torch.float64))
        new = 0.75 * st["mass"] + sums.float().view(-1, page, kv).transpose(1, 2)
        st["out"].copy_(torch.where(seen.view(-1, 1, page), new, st["out"]))
        return st["out"]
    keep, first, recent = case["keep"], case["first"], case["recent"]
    kept = torch.full((len(st["ctx"]), kv, keep), -1, dtype=torch.int32, device="cuda")
    slots = torch.arange(keep, device="cuda")
    for s, (_, n) in enumerate(st["ctx"]):
        at = token_rows(st, s, n)
        to = st["dst"][s, slots // page].long() * page + slots % page
        for h in range(kv):
            if n <= keep:
                ids = torch.arange(n, device="cuda")
            else:
                w = st["mass"][at // page, h, at % page]
                middle = w[first:n - recent]
                best = torch.sort(middle, descending=True, stable=True).indices[:keep - first - recent] + first
                ids = torch.cat([torch.arange(first, device="cuda"), best.sort().values, torch.arange(n - recent, n, device="cuda")])
            kept[s, h, :len(ids)] = ids.int()
            src, dst = at[ids], to[:len(ids)]
            for x in (st["k"], st["v"], st["scale"]):
                if x is not None:
                    flat = x.view(-1, *x.shape[2:])
                    flat[dst, h] = flat[src, h]
            st["mass"][dst // page, h, dst % page] = st["mass"][src // page, h, src % page]
    return moved(st, kept)


# ---- from the definition, in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    heads, kv, dim, page, rows = case["heads"], case["kv"], case["dim"], case["page"], case["rows"]
    share = heads // kv
    pages_of = lambda s, n: st["table"][s, :-(-n // page)].long()
    if case["do"] == "evict":
        kept, ks, vs, cs, ms = [], *(torch.zeros_like(x[st["first_dst"]:]) if x is not None else None for x in (st["k"], st["v"], st["scale"], st["mass"]))
        for s, (_, n) in enumerate(st["ctx"]):
            p = pages_of(s, n)
            m = min(n, case["keep"])
            for h in range(kv):
                w = st["mass"][p, h].reshape(-1)[:n].double().cpu()
                must = torch.zeros(n, dtype=torch.bool)
                must[:case["first"]] = True
                must[n - case["recent"]:] = True
                # by weight, the earlier of equals first; what has to stay goes ahead of everything
                rank = sorted(range(n), key=lambda i: (not bool(must[i]), 0.0 if must[i] else -float(w[i]), i)) if n <= 4096 else None
                if rank is None:
                    key = torch.where(must, torch.full_like(w, float("inf")), w).numpy()
                    import numpy as np
                    rank = np.lexsort((np.arange(n), -key)).tolist()
                ids = sorted(rank[:m])
                row = torch.tensor(ids + [-1] * (case["keep"] - m), dtype=torch.int32)
                kept.append(row)
                i = row[:m].long().cuda()
                j = torch.arange(m, device="cuda")
                to = st["dst"][s].long()[j // page] - st["first_dst"]
                ks[to, j % page, h] = st["k"][p[i // page], i % page, h]
                vs[to, j % page, h] = st["v"][p[i // page], i % page, h]
                ms[to, h, j % page] = st["mass"][p[i // page], h, i % page]
                if cs is not None:
                    cs[to, j % page, h] = st["scale"][p[i // page], i % page, h]
        kept = torch.stack(kept).view(len(st["ctx"]), kv, -1).cuda()
        value = lambda x: x.view(torch.float8_e4m3fn).double() if x.dtype == torch.uint8 else x.double()
        return (kept, value(ks), value(vs), ms.double()) if cs is None else (kept, value(ks), value(vs), cs.double(), ms.double())
    if case["rows"] * sum(n for _, n in st["ctx"]) * heads * dim > 4e11:
        return None
    out, lses = [], []
    total = st["out"].double().clone() if case["do"] == "mass" else None
    first_seen = set()
    for s, (_, n) in enumerate(st["ctx"]):
        p = pages_of(s, n)
        o = torch.empty(rows, heads, dim, dtype=torch.float64, device="cuda")
        l = torch.empty(rows, heads, dtype=torch.float64, device="cuda")
        got = torch.zeros(p.shape[0], kv, page, dtype=torch.float64, device="cuda")
        for h in range(heads):
            keys = st["k"][p, :, h // share].reshape(-1, dim)[:n].double()
            e = (st["q"][s * rows:(s + 1) * rows, h].double() @ keys.t()).mul_(dim ** -0.5)
            for r in range(rows if rows <= 32 else 0):
                e[r, int(n - rows + r + 1):] = -math.inf
            if rows > 32:
                e.masked_fill_(torch.ones_like(e, dtype=torch.bool).triu_(n - rows + 1), -math.inf)
            l[:, h] = torch.logsumexp(e, -1)
            if total is None:
                o[:, h] = torch.softmax(e, -1) @ st["v"][p, :, h // share].reshape(-1, dim)[:n].double()
            else:
                e.sub_((l[:, h] if st["lse"] is None else st["lse"][s * rows:(s + 1) * rows, h].double())[:, None]).exp_()
                w = torch.zeros(p.shape[0] * page, dtype=torch.float64, device="cuda")
                w[:n] = e.sum(0)
                got[:, h // share] += w.view(-1, page)
        if total is None:
            out.append(o.view(rows, -1))
            lses.append(l)
            continue
        for j, pg in enumerate(p.tolist()):
            live = slice(0, min(page, n - j * page))
            if pg not in first_seen:
                first_seen.add(pg)
                total[pg, :, live] = 0.75 * st["mass"][pg, :, live].double()
            total[pg, :, live] += got[j, :, live]
    return total if total is not None else (torch.cat(out), torch.cat(lses))


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    heads, kv, dim, rows = case["heads"], case["kv"], case["dim"], case["rows"]
    ctx, whole = contexts(case), shared_tokens(case)
    if case["do"] == "evict":
        kept = sum(min(n, case["keep"]) for _, n in ctx)
        row = 2 * dim * case["bits"] // 8 + (8 if case["bits"] == 8 else 0) + 4          # keys, values, scales, sum
        return dict(bytes=kv * (2 * kept * row + 4 * sum(n for _, n in ctx) + 4 * case["keep"] * len(ctx)), flops=kv * sum(n for _, n in ctx))
    held = case["groups"] * whole + sum(n - (whole if g is not None else 0) for g, n in ctx)         # tokens, shared ones once
    seen = sum(n - rows + r + 1 for _, n in ctx for r in range(rows))                                # keys, summed over the rows
    T = len(ctx) * rows
    if case["do"] == "attend":
        return dict(bytes=held * kv * dim * 4 + T * heads * (dim * 4 + 4), flops=4 * seen * heads * dim)
    once = 2 * seen * heads * dim
    return dict(bytes=held * kv * (dim * 2 + 8) + T * heads * (dim * 2 + 4), flops=once if rows <= 32 else 2 * once)
