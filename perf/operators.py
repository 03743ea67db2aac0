"""The latent cache of the MLA models in 4 and 8 bits, as calls that can be timed and checked: the step that writes it, its rows read back,
and the attention of decode and verify rows over it.

A token's row holds its normed latent (width L) in codes and its rotated key part (width R) in 16 bits, as bytes of one uint8 row:

* 4 bits: groups of 16 values share a scale of four significant bits, 2^-20 to 1.875 * 2^10, in one byte ((exponent + 20) << 3 | fraction): the
  group's largest magnitude / 7. A code is the nearest whole multiple, -7 to 7, held + 8 in a nibble; of eight values' 32-bit word, nibble i holds value
  2 i and nibble 4 + i value 2 i + 1.
* 8 bits: groups of 32 values share a power of two 2^k (byte k + 127, k from -15 to 7), the smallest that brings the largest magnitude to 448 or
  less; a code is the nearest e4m3 number.
* A group with a value that is no finite number has scale byte 255 and reads back as NaN.

Row: codes | R numbers of 16 bits | scale bytes | zeros up to 16 bytes. Scale bytes go half by half of every 64 values: first those of the lower 32 of
all 64s, then those of the upper 32. Every value of a row (code times scale) is a number of bf16 and of fp16.

The norm and the angles are taken in 64 bits, so that a code is decided by one rounding.
"""
from __future__ import annotations

import math

import torch

own = False

R = 64                       # width of the rotated key part
PAGES = 1.25                 # pages in a pool beyond those in use


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    """`bits` of the cache; `heads` of a rank; `streams` of unequal length, the longest with `context` tokens in its cache; `rows`: new tokens per
    stream (the last ones of its context)."""
    case = lambda name, do, bits, heads, streams, context, rows, latent=512, page=64: dict(
        name=name, do=do, bits=bits, heads=heads, streams=streams, context=context, rows=rows, latent=latent, page=page)
    return [
        # a decode step of a loaded server writes a row per stream, far into their contexts
        case("write-24", "write", 4, 128, 24, 60000, 1),
        # a chunk of a prompt is written
        case("write-2048", "write", 8, 128, 1, 2048, 2048),
        case("write-1111", "write", 4, 32, 1, 5000, 1111),
        # a prompt's next chunk takes back all of the conversation so far; two prompts that share a step
        case("read-13111", "read", 4, 128, 1, 13111, 1111),
        case("read-2", "read", 8, 128, 2, 5003, 900),
        # one stream decodes: latency
        case("attend-1", "attend", 4, 128, 1, 2048, 1),
        # a long document behind one stream
        case("attend-1-long", "attend", 4, 128, 1, 100000, 1),
        # several users at once, in both formats
        case("attend-6", "attend", 4, 128, 6, 4000, 1),
        case("attend-6-fp8", "attend", 8, 128, 6, 4000, 1),
        # a loaded server
        case("attend-24", "attend", 4, 128, 24, 16000, 1),
        # the same on a rank of eight that holds an eighth of the heads
        case("attend-32-rank", "attend", 4, 16, 32, 16000, 1),
        # drafted tokens verified on such a rank
        case("attend-verify", "attend", 8, 16, 2, 8000, 17),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    do, bits, page = rng.choice(["write", "read", "attend", "attend", "attend"]), rng.choice([4, 4, 8]), rng.choice([64, 64, 128, 32])
    latent = rng.choice([512, 512, 512, 128, 64])
    heads = rng.choice([128, 64, 32, 16, 8, 4, 20]) if latent == 512 else rng.choice([4, 6, 16])
    if do == "write":
        rows = rng.choice([1, log(2, 32), log(33, 2048)])
        streams = log(1, 48) if rows == 1 else log(1, 4)
        context = max(rows, log(64, 60000))
    elif do == "read":
        streams, context = log(1, 4), log(40, 30000)
        context = max(1, context // streams)
        rows = min(context, log(33, 2048))
    else:
        rows = rng.choice([1, 1, log(2, 20)])
        streams = log(1, 48 if rows == 1 else 6)
        context = max(rows, log(1, 24 * 16000 * 128 // (heads * streams * rows)))
        context = min(context, 100000 // max(1, streams // 4))
    return dict(do=do, bits=bits, heads=heads, streams=streams, context=context, rows=rows, latent=latent, page=page)


def lengths(case):
    """Tokens in every stream's cache with the new ones."""
    return [max(case["rows"], int(case["context"] * (1 - 0.7 * ((i * 0.618) % 1)))) for i in range(case["streams"])]


def row_bytes(latent, bits):
    codes, scales = latent * bits // 8, latent // (16 if bits == 4 else 32)
    return (codes + 2 * R + scales + 15) // 16 * 16


def scale_order(latent, bits):
    """Where the scale byte of every group lies: position -> group."""
    per = 2 if bits == 4 else 1                          # groups in 32 values
    return [chunk * 2 * per + half * per + j for half in range(2) for chunk in range(latent // 64) for j in range(per)]


# ---- the plain form: rows of bytes ------------------------------------------------------------------------------------

def significant(x, digits):
    """x in 64 bits, rounded to `digits` binary digits (halves to the even one)."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 2.0 ** digits), e - digits)


def quantise(y, bits):
    """y [rows, L] in 64 bits -> codes as whole numbers or e4m3 values [rows, L], scales [rows, groups], scale bytes."""
    size = 16 if bits == 4 else 32
    g = y.view(y.shape[0], -1, size)
    bad = ~torch.isfinite(g).all(-1)
    top = torch.where(bad[..., None], torch.zeros_like(g), g).abs().amax(-1)
    if bits == 4:
        scale = significant(top / 7, 4).clamp(2.0 ** -20, 1.875 * 2.0 ** 10)
        m, e = torch.frexp(scale)                         # scale = (8 + fraction) / 16 * 2^e
        byte = (e.long() + 19) * 8 + torch.round(m * 16).long() - 8
        code = torch.round(g / scale[..., None]).clamp(-7, 7)
    else:
        m, e = torch.frexp(top / 448)
        k = torch.where(m > 0.5, e, e - 1).clamp(-15, 7)
        k = torch.where(top > 0, k, torch.full_like(k, -15))
        scale, byte = torch.ldexp(torch.ones_like(top), k), k.long() + 127
        v = g / scale[..., None]
        step = torch.ldexp(torch.ones_like(v), (torch.frexp(v).exponent - 1).clamp(-6, 8) - 3)
        code = (torch.round(v / step) * step).clamp(-448, 448)
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    return code.view_as(y), scale, torch.where(bad, torch.full_like(byte, 255), byte)


def pack(y, rope, bits):
    """Normed latents [rows, L] (64 bits) and rotated key parts [rows, R] -> the rows' bytes."""
    rows, L = y.shape
    code, _, byte = quantise(y, bits)
    if bits == 4:
        n = (code.long() + 8).view(rows, L // 8, 4, 2)                       # value 2 i + j of a word
        n = torch.cat([n[..., 0], n[..., 1]], -1)                            # nibbles 0..7
        codes = (n[..., 0::2] + 16 * n[..., 1::2]).to(torch.uint8).reshape(rows, -1)
    else:
        codes = code.float().to(torch.float8_e4m3fn).view(torch.uint8)
    parts = [codes, rope.to(torch.bfloat16).contiguous().view(torch.uint8), byte[:, scale_order(L, bits)].to(torch.uint8)]
    out = torch.zeros(rows, row_bytes(L, bits), dtype=torch.uint8, device=y.device)
    at = torch.cat(parts, 1)
    out[:, :at.shape[1]] = at
    return out


def unpack(raw, L, bits):
    """The rows' bytes -> [rows, L + R] in 32 bits."""
    rows, n = raw.shape[0], L * bits // 8
    order = torch.tensor(scale_order(L, bits), device=raw.device)
    scales = L // (16 if bits == 4 else 32)
    byte = torch.empty(rows, scales, dtype=torch.long, device=raw.device)
    byte[:, order] = raw[:, n + 2 * R:n + 2 * R + scales].long()
    if bits == 4:
        b = raw[:, :n].view(rows, L // 8, 4).long()
        nib = torch.stack([b & 15, b >> 4], -1).view(rows, L // 8, 8)
        code = torch.stack([nib[..., :4], nib[..., 4:]], -1).reshape(rows, -1, 16).float() - 8
        scale = torch.ldexp(1 + (byte & 7).float() / 8, (byte >> 3) - 20)
        nan = byte >= 248
    else:
        code = raw[:, :n].contiguous().view(torch.float8_e4m3fn).float().view(rows, -1, 32)
        scale = torch.ldexp(torch.ones(byte.shape, device=raw.device), byte - 127)
        nan = byte >= 135
    v = torch.where(nan[..., None], torch.full_like(code, float("nan")), code * scale[..., None]).view(rows, L)
    return torch.cat([v, raw[:, n:n + 2 * R].contiguous().view(torch.bfloat16).float()], 1)


def normed(kva, w, L, eps):
    x = kva[:, :L].double()
    return x * (1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)) * (1 + w.double())


def rotated(x, pos, inv_freq):
    """Pairs (i, i + R / 2) of the last axis turned by pos * inv_freq[i]; 64 bits."""
    ang = (pos.double()[:, None] * inv_freq.double()[None]).view(pos.shape[0], *([1] * (x.dim() - 2)), R // 2)
    a, b = x[..., :R // 2].double(), x[..., R // 2:].double()
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)


def flat_rows(state, slots, positions):
    """Numbers of the cache rows of (slot, position) pairs."""
    page = state["case"]["page"]
    return state["table"][slots, positions // page].long() * page + positions % page


# ---- inputs ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    """What the engine has in hand: the paged cache with every stream's context in it, the step's tables, its projections (write) or absorbed queries
    (attend). Latents as they come out of a projection: normal, a few channels several times as large as the others, norm weights around one."""
    g = torch.Generator("cuda").manual_seed(seed * 6151 + 17)
    dev, L, bits, page = "cuda", case["latent"], case["bits"], case["page"]
    bf = lambda *s, sc=1.0: (torch.randn(*s, generator=g, device=dev) * sc).to(torch.bfloat16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    lens, rows, heads = lengths(case), case["rows"], case["heads"]
    per = (max(lens) + page - 1) // page
    used = sum((n + page - 1) // page for n in lens)
    order = torch.randperm(int(used * PAGES) + 1, generator=g, device=dev).int()
    table, at = torch.full((len(lens), per), -1, dtype=torch.int32, device=dev), 0
    for s, n in enumerate(lens):
        k = (n + page - 1) // page
        table[s, :k] = order[at:at + k]
        at += k
    st = dict(case=case, table=table, w=bf(L, sc=0.2), inv_freq=(1e4 ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2))).float().to(dev))
    loud = 1 + 7 * (torch.rand(L + R, generator=g, device=dev) < 0.02)
    T = len(lens) * rows
    st["row_slot"] = i32([s for s in range(len(lens)) for _ in range(rows)])
    st["row_pos"] = i32([n - rows + r for n in lens for r in range(rows)])
    st["row_kvlen"] = st["row_pos"] + 1
    st["seg_slot"], st["seg_row0"] = i32(list(range(len(lens)))), i32([s * rows for s in range(len(lens))])
    st["seg_pos0"], st["seg_nrows"] = i32([n - rows for n in lens]), i32([rows] * len(lens))
    cache = torch.empty(order.shape[0] * page, row_bytes(L, bits), dtype=torch.uint8, device=dev)
    for lo in range(0, cache.shape[0], 1 << 16):                              # what other streams left behind lies between
        n = min(1 << 16, cache.shape[0] - lo)
        kva = (torch.randn(n, L + R, generator=g, device=dev) * loud).to(torch.bfloat16)
        cache[lo:lo + n] = pack(normed(kva, st["w"], L, 1e-6), kva[:, L:], bits)
    st["cache"] = cache.view(-1, page, cache.shape[1])
    if case["do"] == "write":
        st["kva"] = (torch.randn(T, L + R, generator=g, device=dev) * loud).to(torch.bfloat16)
        st["dn"] = 128 if L == 512 else 32
        st["q"] = bf(T, heads * (st["dn"] + R))
    if case["do"] == "attend":
        st["scale"] = (L + R) ** -0.5
        st["q"] = bf(T, heads, L + R, sc=1.3)
    if own:
        from ferrite_b200.ops.cuda_ops import CudaOps
        st["ops"] = CudaOps(dev)
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(st):
    return run_own(st) if own else run_plain(st)


def run_own(st):
    case, ops = st["case"], st["ops"]
    L, page, bits, heads = case["latent"], case["page"], case["bits"], case["heads"]
    if case["do"] == "write":
        # the cache rows of the step's tokens; the queries' rotated parts; what the rows stand for
        q = ops.mla_prep(st["q"], st["kva"], st["w"], None, st["inv_freq"], st["row_slot"], st["row_pos"], st["table"], st["cache"], page, heads,
                         st["dn"], L, R, 1e-6, absorb=False, kv_bits=bits)
        rows = ops.mla_rows(st["cache"], st["seg_slot"], st["seg_pos0"], st["seg_nrows"], st["table"], page, L, R, len(st["kva"]), kv_bits=bits)
        return q[:, :, L:], rows
    if case["do"] == "read":
        # every segment's context from the first token on, segment after segment on whole pages, zeros behind the last token of each
        total = sum((n + page - 1) // page * page for n in lengths(case))
        return ops.mla_rows(st["cache"], st["seg_slot"], st["seg_pos0"], st["seg_nrows"], st["table"], page, L, R, total, whole=True, kv_bits=bits)
    segs = (st["seg_slot"], st["seg_row0"], st["seg_nrows"], case["rows"])
    return ops.mla_attention(st["q"], st["cache"], st["row_slot"], st["row_kvlen"], st["table"], page, heads, L, R, st["scale"], segs=segs, kv_bits=bits)


def run_plain(st):
    case = st["case"]
    L, page, bits, heads, rows = case["latent"], case["page"], case["bits"], case["heads"], case["rows"]
    raw = st["cache"].view(-1, st["cache"].shape[-1])
    if case["do"] == "write":
        rope = rotated(st["kva"][:, L:], st["row_pos"], st["inv_freq"])
        at = flat_rows(st, st["row_slot"].long(), st["row_pos"].long())
        raw[at] = pack(normed(st["kva"], st["w"], L, 1e-6), rope, bits)
        q = rotated(st["q"].view(len(at), heads, -1)[..., st["dn"]:], st["row_pos"], st["inv_freq"])
        return q.to(torch.bfloat16), unpack(raw[at], L, bits).to(torch.bfloat16)
    outs = []
    for s, n in enumerate(lengths(case)):
        at = flat_rows(st, torch.full((n,), s, device=raw.device), torch.arange(n, device=raw.device))
        keys = unpack(raw[at], L, bits)
        if case["do"] == "read":
            outs.append(keys.to(torch.bfloat16))
            outs.append(keys.new_zeros((-n) % page, L + R).to(torch.bfloat16))
            continue
        sc = (st["q"][s * rows:(s + 1) * rows].float() @ keys.t()) * st["scale"]                 # [rows, heads, n]
        sees = torch.arange(n, device=raw.device)[None, None] < st["row_kvlen"][s * rows:(s + 1) * rows, None, None]
        sc = torch.where(sees, sc, torch.full_like(sc, float("-inf")))
        p = (sc - sc.amax(-1, keepdim=True)).exp()
        outs.append(((p / p.sum(-1, keepdim=True)) @ keys[:, :L]).to(torch.bfloat16))
    return torch.cat(outs)


# ---- from the definition, in 64 bits --------------------------------------------------------------------------------

def value_of(raw, L, bits):
    """[rows, L + R] in 64 bits, value by value from the description of a row at the top."""
    rows, n = raw.shape[0], L * bits // 8
    e = torch.arange(L, device=raw.device)
    per = 2 if bits == 4 else 1
    at = n + 2 * R + (e % 64 // 32) * (L // 64 * per) + e // 64 * per + (e % 32 // 16 if bits == 4 else 0)
    byte = raw[:, at].int()
    if bits == 4:
        nibble = e % 8 // 2 + 4 * (e % 2)                                       # of the value's word
        held = (raw[:, e // 8 * 4 + nibble // 2].int() >> (nibble % 2 * 4).int()) & 15
        v = (held - 8).double() * (8 + byte % 8).double() * torch.pow(2.0, (byte // 8 - 23).double())
    else:
        c = raw[:, :n].int()
        ex, fr = c // 8 % 16, (c % 8).double()
        v = torch.where(ex > 0, (8 + fr) * torch.pow(2.0, (ex - 10).double()), fr * 2.0 ** -9) * torch.where(c > 127, -1.0, 1.0)
        v = v * torch.pow(2.0, (byte - 127).double())
    return torch.cat([v, raw[:, n:n + 2 * R].contiguous().view(torch.bfloat16).double()], 1)


def nearest(y, bits):
    """y rounded to what its group can hold, by trying: the scale from its own definition, the code as the closest of all."""
    rows, L = y.shape
    size = 16 if bits == 4 else 32
    g = y.reshape(-1, size)
    top = g.abs().max(1, keepdim=True).values
    if bits == 4:
        steps = torch.tensor([(8 + f) * 2.0 ** (e - 3) for e in range(-20, 11) for f in range(8)], dtype=torch.float64, device=y.device)
        held = torch.arange(-7, 8, dtype=torch.float64, device=y.device)
        at = torch.searchsorted(steps, (top / 7).contiguous()).clamp(1, len(steps) - 1)
        lo, hi = steps[at - 1], steps[at]
        scale = torch.where(top / 7 - lo <= hi - top / 7, torch.where((top / 7 - lo == hi - top / 7) & (at % 2 == 0), hi, lo), hi)
    else:
        half = [f * 2.0 ** -9 for f in range(8)] + [(8 + f) * 2.0 ** (e - 10) for e in range(1, 16) for f in range(8) if not (e == 15 and f == 7)]
        held = torch.tensor(sorted({-v for v in half} | set(half)), dtype=torch.float64, device=y.device)
        scale = torch.pow(2.0, torch.arange(-15, 8, dtype=torch.float64, device=y.device))
        scale = scale[torch.searchsorted(448 * scale, top.contiguous()).clamp(0, 22)]
    mid = (held[1:] + held[:-1]) / 2
    return (held[torch.searchsorted(mid, (g / scale).contiguous())] * scale).view(rows, L)


def exact(case, seed):
    st = prepare(case, seed)
    L, bits, rows, heads, page = case["latent"], case["bits"], case["rows"], case["heads"], case["page"]
    raw = st["cache"].view(-1, st["cache"].shape[-1])
    turn = lambda x, pos: torch.view_as_real(torch.complex(x[..., :R // 2].double(), x[..., R // 2:].double()) * torch.polar(
        torch.ones((), dtype=torch.float64, device=x.device), pos.double().view(-1, *([1] * (x.dim() - 1))) * st["inv_freq"].double())).transpose(-1, -2).flatten(-2)
    if case["do"] == "write":
        x = st["kva"][:, :L].double()
        y = x / (x.square().sum(1, keepdim=True) / L + 1e-6).sqrt() * (1 + st["w"].double())
        q = turn(st["q"].view(len(x), heads, -1)[..., st["dn"]:], st["row_pos"])
        return q, torch.cat([nearest(y, bits), turn(st["kva"][:, L:], st["row_pos"])], 1)
    outs = []
    for s, n in enumerate(lengths(case)):
        pages = st["table"][s, :(n + page - 1) // page].long()
        keys = value_of(st["cache"][pages].view(-1, raw.shape[1]), L, bits)
        if case["do"] == "read":
            outs.append(torch.cat([keys[:n], torch.zeros_like(keys[n:])]))
            continue
        for r in range(rows):
            k = keys[:n - rows + r + 1]
            p = torch.softmax(st["q"][s * rows + r].double() @ k.t() * st["scale"], -1)
            outs.append((p @ k[:, :L])[None])
    return torch.cat(outs)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    L, bits, rows, heads = case["latent"], case["bits"], case["rows"], case["heads"]
    held = L * bits // 8 + L // (16 if bits == 4 else 32) + 2 * R                  # bytes of a row that say something
    lens = lengths(case)
    T = len(lens) * rows
    if case["do"] == "write":
        # projections and query parts in, cache rows out and in again, query parts and the rows' values out
        return dict(bytes=T * ((L + R) * 2 + heads * R * 4 + 2 * held + (L + R) * 2) + L * 2, flops=T * (8 * L + 3 * R * (heads + 1)))
    if case["do"] == "read":
        return dict(bytes=sum(n * held + (n + case["page"] - 1) // case["page"] * case["page"] * (L + R) * 2 for n in lens), flops=sum(lens) * L)
    seen = sum(n - rows + r + 1 for n in lens for r in range(rows))                # keys, summed over the rows
    return dict(bytes=sum(lens) * held + T * heads * (2 * L + R) * 2, flops=2 * seen * heads * (2 * L + R))
