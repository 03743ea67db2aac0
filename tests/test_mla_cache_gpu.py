"""Latent cache of the MLA models in 4 and 8 bits on the GPU: the step that writes it, its rows read back and the attention over it against the plain
statement in 64 bits (`latent_rows.py`), alone and as the engine runs them."""
import functools
import sys
import zlib

import latent_rows as lr
import pytest
import torch

from ferrite_b200.ops import mla_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"
R = 64
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.fixture(scope="module")
def ops(ext):
    from ferrite_b200.ops.cuda_ops import CudaOps
    return CudaOps(DEV)


@pytest.fixture(autouse=True)
def clean(request):
    yield
    if "ops" in request.fixturenames:
        o = request.getfixturevalue("ops")
        assert o.status() == 0


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(key).encode()))


def bf(g, *s, sc=1.0):
    return (torch.randn(*s, generator=g, device=DEV) * sc).to(torch.bfloat16)


def tables(lens, page, g, spare=3, width=0):
    """Pages of every stream in no order, -1 behind them, and the number of pages of the pool."""
    need = [(n + page - 1) // page for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device=DEV).int()
    t = torch.full((len(lens), max(max(need), 1) + width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, k in enumerate(need):
        t[s, :k] = order[at:at + k]
        at += k
    return t, total


def inv_freq():
    return (1e4 ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2))).float().to(DEV)


def prep(ops, bits, L, nq, dn, slot, pos, table, pages, page, g, kva=None, cache=None, q=None):
    T = len(slot)
    kva = bf(g, T, L + R) if kva is None else kva
    q = bf(g, T, nq * (dn + R)) if q is None else q
    w = bf(g, L, sc=0.2)
    cache = torch.randint(0, 256, (pages, page, lr.row_bytes(L, bits)), generator=g, device=DEV, dtype=torch.uint8) if cache is None else cache
    before = cache.clone()
    got = ops.mla_prep(q, kva, w, None, inv_freq(), i32(slot), i32(pos), table, cache, page, nq, dn, L, R, 1e-6, absorb=False, kv_bits=bits)
    return got, cache, before, q, kva, w


def check_prep(bits, L, nq, dn, slot, pos, table, page, got, cache, before, q, kva, w):
    flat = [int(table[s, p // page]) * page + p % page for s, p in zip(slot, pos)]
    raw = cache.view(-1, cache.shape[-1])
    vals = lr.unpack(raw[flat], L, bits)
    p = torch.tensor(pos, device=DEV)
    y = lr.normed(kva, w, L, 1e-6)
    assert torch.equal(vals[:, :L].nan_to_num(99), mla_cache.quantised(y, bits).cpu().nan_to_num(99))       # decided by one rounding of the exact value
    # one rounding to bf16 (2^-8 of the value) and sines and cosines in 32 bits (a few 2^-24 of what they multiply)
    key = kva[:, L:L + R].double()
    ext = (key[:, :32].abs() + key[:, 32:].abs()).repeat(1, 2)
    want = lr.rotated(kva[:, L:L + R], p, inv_freq())
    assert ((vals[:, L:].to(DEV) - want).abs() <= 2 ** -8 * want.abs() + 2 ** -20 * ext).all()
    qr = q.reshape(len(slot), nq, dn + R)[..., dn:]
    want = lr.rotated(qr, p, inv_freq())
    ext = (qr[..., :32].double().abs() + qr[..., 32:].double().abs()).repeat(1, 1, 2)
    assert ((got[..., L:].double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -20 * ext).all()
    n = lr.R * 2 + L * bits // 8 + L // (16 if bits == 4 else 32)
    assert not raw[flat][:, n:].any()                                                                    # zeros up to 16 bytes
    rest = torch.ones(raw.shape[0], dtype=torch.bool, device=DEV)
    rest[flat] = False
    assert torch.equal(raw[rest], before.view(-1, cache.shape[-1])[rest])                                 # nothing else moved


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("L,nq,dn,page", [(512, 128, 128, 64), (512, 5, 128, 16), (64, 4, 32, 64), (192, 33, 20, 1), (256, 1, 0, 40)])
@pytest.mark.parametrize("rows", [1, 7, 300])
def test_prep_writes_rows(ops, bits, L, nq, dn, page, rows):
    g = gen("prep", bits, L, nq, rows)
    lens = [rows + 70001, 130]
    slot, pos = [0] * rows + [1] * 2, list(range(70001, 70001 + rows)) + [0, 129]
    table, pages = tables(lens, page, g)
    args = prep(ops, bits, L, nq, dn, slot, pos, table, pages, page, g)
    check_prep(bits, L, nq, dn, slot, pos, table, page, *args)


@pytest.mark.parametrize("bits", [4, 8])
def test_prep_of_unusual_rows(ops, bits):
    """Rows of zeros, tiny, huge and ragged ones, values that are no numbers; strides; the same call again gives the same bytes."""
    L, nq, dn, page, T = 512, 3, 128, 64, 12
    g = gen("odd", bits)
    wide = bf(g, T, L + R + 24)
    kva = wide[:, 8:8 + L + R]
    kva[0] = 0
    kva[1] *= 1e-30
    kva[2] *= 1e30
    kva[3, ::17] *= 3000
    kva[4, 40] = float("nan")
    kva[5, 100] = float("inf")
    kva[6, :L] = 1.0
    kva[7, 1:L] = 0
    q = bf(g, T, nq * (dn + R) + 3)[:, 3:]                                                                # rows on no 8 bytes
    table, pages = tables([T], page, g)
    slot, pos = [0] * T, list(range(T))
    args = prep(ops, bits, L, nq, dn, slot, pos, table, pages, page, g, kva=kva, q=q)
    check_prep(bits, L, nq, dn, slot, pos, table, page, *args)
    again = args[1].clone()
    ops.mla_prep(q, kva, args[-1], None, inv_freq(), i32(slot), i32(pos), table, again, page, nq, dn, L, R, 1e-6, absorb=False, kv_bits=bits)
    assert torch.equal(again, args[1])


def random_cache(bits, L, pages, page, g):
    """A cache as prep leaves it, written by the plain quantiser's own values through the kernel: rows of normal latents."""
    raw = torch.randint(0, 256, (pages, page, lr.row_bytes(L, bits)), generator=g, device=DEV, dtype=torch.uint8)
    n = L * bits // 8
    if bits == 8:
        raw[..., :n] = torch.where(raw[..., :n] & 127 == 127, raw[..., :n] - 1, raw[..., :n])            # e4m3 has no number there
    raw[..., n:n + 2 * R] = bf(g, pages, page, R, sc=2.0).view(torch.uint8).view(pages, page, 2 * R)
    ns = L // (16 if bits == 4 else 32)
    lo, hi = ((20 - 5) * 8, (20 - 1) * 8) if bits == 4 else (127 - 9, 127 - 7)                             # values of about one
    raw[..., n + 2 * R:n + 2 * R + ns] = torch.randint(lo, hi, (pages, page, ns), generator=g, device=DEV, dtype=torch.uint8)
    return raw


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("L,page", [(512, 64), (512, 24), (64, 64), (320, 128)])
def test_rows_read_back(ops, bits, L, page):
    g = gen("rows", bits, L, page)
    lens, rows = [1, 200, 64, 129], [1, 37, 64, 0]
    table, pages = tables(lens, page, g)
    cache = random_cache(bits, L, pages, page, g)
    vals = lr.unpack(cache.view(-1, cache.shape[-1]), L, bits)
    at = lambda s, p: int(table[s, p // page]) * page + p % page
    seg = i32([0, 1, 2, 3]), i32([n - r for n, r in zip(lens, rows)]), i32(rows)
    got = ops.mla_rows(cache, *seg, table, page, L, R, sum(rows) + 5, kv_bits=bits).cpu().double()
    want = vals[[at(s, p) for s in range(4) for p in range(lens[s] - rows[s], lens[s])]]
    assert torch.equal(got[:len(want)], want) and not got[len(want):].any()
    total = sum((n + page - 1) // page * page for n in lens)
    got = ops.mla_rows(cache, *seg, table, page, L, R, total, whole=True, kv_bits=bits).cpu().double()
    lo = 0
    for s, n in enumerate(lens):
        hi = lo + (n + page - 1) // page * page
        assert torch.equal(got[lo:lo + n], vals[[at(s, p) for p in range(n)]]) and not got[lo + n:hi].any()
        lo = hi
    assert ops.mla_rows(cache, *seg, table, page, L, R, 0, kv_bits=bits).shape == (0, L + R)


def test_rows_say_which_groups_are_no_numbers(ops):
    g = gen("nan")
    for bits in (4, 8):
        cache = random_cache(bits, 128, 1, 64, g)
        cache[0, 7, 128 * bits // 8 + 2 * R] = 255
        got = ops.mla_rows(cache, i32([0]), i32([0]), i32([64]), i32([[0]]), 64, 128, R, 64, kv_bits=bits)
        bad = torch.zeros(64, 192, dtype=torch.bool, device=DEV)
        bad[7, :mla_cache.GROUP[bits]] = True
        assert torch.equal(got.isnan(), bad)


def check_attention(ops, bits, L, nq, page, slot, kvlen, table, cache, q, scale, segs=None):
    """Off 64 bits by: the rounding of the result to bf16, 2^-8 of it; softmax weights of 11 bits, 2^-11 of the weighted mean of |value|; scores summed
    in 32 bits over L + R products in steps of 16 (each 2^-23 of the sum of magnitudes), which move a weight by as much of itself, twice."""
    got = ops.mla_attention(q, cache, i32(slot), i32(kvlen), table, page, nq, L, R, scale, segs=segs, kv_bits=bits)
    vals = lr.unpack(cache.view(-1, cache.shape[-1]), L, bits).to(DEV)
    for r, (s, n) in enumerate(zip(slot, kvlen)):
        p = torch.arange(n, device=DEV)
        keys = vals[table[s, p // page].long() * page + p % page]
        qr = q[r].double()
        want = lr.attend(qr, keys, L, scale)
        if n == 0:
            assert not got[r].any()
            continue
        w = torch.softmax(qr @ keys.t() * scale, -1)
        mean = w @ keys[:, :L].abs()
        ds = (qr.abs() @ keys.abs().t() * scale).amax(-1, keepdim=True) * (L + R) / 16 * 2 ** -23
        tol = 2 ** -8 * want.abs() + mean * (2 ** -11 + 2 * ds) + 1e-30
        off = (got[r].double() - want).abs()
        assert (off <= tol).all(), (r, n, (off / tol).max().item())
    return got


def segments(rows, n):
    return i32(list(range(n))), i32([s * rows for s in range(n)]), i32([rows] * n), rows


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("L,nq", [(512, 128), (512, 16), (512, 3), (256, 20), (128, 32), (64, 4)])
@pytest.mark.parametrize("lens,rows,page", [((1, 127, 128, 129, 64), 1, 64), ((1000, 300), 5, 64), ((200,), 40, 24), ((5000,), 1, 128), ((700, 30), 17, 64)])
def test_attention(ops, bits, L, nq, lens, rows, page):
    g = gen("attn", bits, L, nq, rows, page)
    table, pages = tables(lens, page, g)
    cache = random_cache(bits, L, pages, page, g)
    slot = [s for s in range(len(lens)) for _ in range(rows)]
    kvlen = [max(1, n - rows + 1 + r) for n in lens for r in range(rows)]
    q = bf(g, len(slot), nq, L + R)
    scale = (L + R) ** -0.5
    got = check_attention(ops, bits, L, nq, page, slot, kvlen, table, cache, q, scale, segments(rows, len(lens)))
    alone = check_attention(ops, bits, L, nq, page, slot, kvlen, table, cache, q, scale)                       # without segments: every row one of its own
    if rows == 1:
        assert torch.equal(got, alone)


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_of_rows_that_see_nothing(ops, bits):
    g = gen("none", bits)
    table, pages = tables([100, 100, 100], 64, g)
    cache = random_cache(bits, 512, pages, 64, g)
    q = bf(g, 3, 16, 576)
    check_attention(ops, bits, 512, 16, 64, [0, 1, 2], [0, 77, 0], table, cache, q, 0.05, segments(1, 3))
    assert ops.mla_attention(q[:0], cache, i32([]), i32([]), table, 64, 16, 512, R, 0.05, kv_bits=bits).shape == (0, 16, 512)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nq", [128, 24, 8])
def test_attention_with_scores_that_grow(ops, bits, nq):
    """Scores far apart and rising along the keys, so that the running maximum moves again and again; and far below zero throughout."""
    g = gen("grow", bits, nq)
    n, L = 900, 512
    table, pages = tables([n, n], 64, g)
    cache = random_cache(bits, L, pages, 64, g)
    at = L * bits // 8
    ramp = torch.linspace(0, 60, n, device=DEV).to(torch.bfloat16)
    rope = torch.zeros(n, R, dtype=torch.bfloat16, device=DEV)
    rope[:, 0] = ramp
    for s in range(2):
        p = torch.arange(n, device=DEV)
        flat = table[s, p // 64].long() * 64 + p % 64
        cache.view(-1, cache.shape[-1])[flat, at:at + 2 * R] = (rope if s == 0 else rope - 70).view(torch.uint8).view(n, 2 * R)
    q = bf(g, 2, nq, L + R, sc=0.2)
    q[..., L] = 100
    check_attention(ops, bits, L, nq, 64, [0, 1], [n, n], table, cache, q, 0.05, segments(1, 2))


@pytest.mark.parametrize("bits", [4, 8])
def test_attention_scales_of_queries(ops, bits):
    """Queries of any size: tiny, large, zero, one loud value beside small ones."""
    g = gen("scale", bits)
    table, pages = tables([300], 64, g)
    cache = random_cache(bits, 512, pages, 64, g)
    q = bf(g, 1, 20, 576)
    q[0, 0] *= 1e-20
    q[0, 1] = 0
    q[0, 2] *= 20
    q[0, 3, 17] = 200
    q[0, 4, 520] = -300
    q[0, 5, :512] *= 1e-6
    check_attention(ops, bits, 512, 20, 64, [0], [300], table, cache, q, 0.05, segments(1, 1))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nq", [128, 16])
def test_values_that_are_no_numbers_reach_who_sees_them(ops, bits, nq):
    """A row whose latent is no number is seen by the rows at and behind it alone; queries that are none spoil their head alone; what lies behind the
    context, in its last page and tile too, is no matter."""
    g = gen("poison", bits, nq)
    L, n, rows = 512, 200, 6
    table, pages = tables([n], 64, g)
    cache = random_cache(bits, L, pages, 64, g)
    raw = cache.view(-1, cache.shape[-1])
    at = lambda p: int(table[0, p // 64]) * 64 + p % 64
    for p in range(n, (n + 63) // 64 * 64):
        raw[at(p)] = 255
    q = bf(g, rows, nq, L + R)
    kvlen = [n - rows + 1 + r for r in range(rows)]
    clean = check_attention(ops, bits, L, nq, 64, [0] * rows, kvlen, table, cache, q, 0.05, segments(rows, 1))
    raw[at(n - 3), L * bits // 8 + 2 * R + 5] = 255                                                # seen by the last three rows
    q[1, 2, 100] = float("nan")
    q[0, 3, 570] = float("inf")
    got = ops.mla_attention(q, cache, i32([0] * rows), i32(kvlen), table, 64, nq, L, R, 0.05, segs=segments(rows, 1), kv_bits=bits)
    bad = torch.zeros(rows, nq, dtype=torch.bool, device=DEV)
    bad[3:] = True
    bad[1, 2] = bad[0, 3] = True
    assert torch.equal(got.isnan().all(-1), bad) and torch.equal(got.isnan().any(-1), bad)
    assert torch.equal(got[~bad], clean[~bad])


def test_refusals(ops):
    g = gen("no")
    table, pages = tables([64], 64, g)
    c4 = random_cache(4, 512, pages, 64, g)
    q = bf(g, 1, 16, 576)
    call = lambda q=q, cache=c4, slot=i32([0]), kvlen=i32([64]), t=table, page=64, L=512, bits=4: ops.mla_attention(
        q, cache, slot, kvlen, t, page, q.shape[1], L, R, 0.05, kv_bits=bits)
    call()
    for kw in (dict(bits=8), dict(bits=6), dict(page=32), dict(L=448), dict(cache=c4.float()), dict(t=table.long()), dict(slot=i32([0, 0])),
               dict(kvlen=i32([64]).long()), dict(q=q.float()), dict(cache=c4[:, :, :400]), dict(t=table.cpu())):
        with pytest.raises(RuntimeError):
            call(**kw)
    rows = lambda cache=c4, seg=i32([0]), L=512, bits=4: ops.mla_rows(cache, seg, i32([0]), i32([64]), table, 64, L, R, 64, kv_bits=bits)
    rows()
    for kw in (dict(bits=8), dict(L=256), dict(seg=i32([0, 0])), dict(cache=c4.to(torch.int8))):
        with pytest.raises(RuntimeError):
            rows(**kw)
    put = lambda cache=c4, kva=bf(g, 1, 576), q=bf(g, 1, 16 * 192), w=bf(g, 512), pos=i32([3]), dn=128, bits=4: ops.mla_prep(
        q, kva, w, None, inv_freq(), i32([0]), pos, table, cache, 64, 16, dn, 512, R, 1e-6, absorb=False, kv_bits=bits)
    put()
    for kw in (dict(bits=8), dict(kva=bf(g, 1, 570)), dict(kva=bf(g, 2, 576)), dict(w=bf(g, 64)), dict(pos=i32([3]).long()), dict(dn=126), dict(q=bf(g, 1, 5)),
               dict(kva=bf(g, 1, 576).float())):
        with pytest.raises(RuntimeError):
            put(**kw)


def test_pages_that_are_not_there_set_the_status(ops):
    g = gen("pages")
    table, pages = tables([128], 64, g)
    cache = random_cache(4, 512, pages, 64, g)
    bad = table.clone()
    q = bf(g, 1, 16, 576)
    for entry in (-1, pages, pages + 1000):
        bad[0, 1] = entry
        for call in (lambda: ops.mla_attention(q, cache, i32([0]), i32([128]), bad, 64, 16, 512, R, 0.05, kv_bits=4),
                     lambda: ops.mla_rows(cache, i32([0]), i32([0]), i32([128]), bad, 64, 512, R, 128, kv_bits=4),
                     lambda: prep(ops, 4, 512, 16, 128, [0], [100], bad, pages, 64, g, cache=cache)):
            before = cache.clone()
            call()
            assert ops.status() == 3 and torch.equal(cache, before)
            ops.status_word.zero_()
    # a length beyond the table
    ops.mla_attention(q, cache, i32([0]), i32([200]), table, 64, 16, 512, R, 0.05, kv_bits=4)
    assert ops.status() == 3
    ops.status_word.zero_()


@pytest.mark.parametrize("bits", [4, 8])
def test_write_attend_and_read_back_as_a_prompt_and_a_decode_step_do(ops, bits):
    """A prompt's rows are written and its expanded attention reads them back; a decode row behind it is written and attends. Both against 64 bits over
    the values that the cache holds."""
    L, nq, dn, dv, page, n = 512, 16, 128, 128, 64, 150
    g = gen("run", bits)
    table, pages = tables([n + 1], page, g)
    cache = torch.zeros(pages, page, lr.row_bytes(L, bits), dtype=torch.uint8, device=DEV)
    w, w_uk, w_uv = bf(g, L, sc=0.2), bf(g, nq, L, dn, sc=dn ** -0.5), bf(g, nq, dv, L, sc=L ** -0.5)
    kv_b = torch.cat([w_uk.transpose(1, 2), w_uv], 1).reshape(nq * (dn + dv), L).contiguous()
    q, kva = bf(g, n + 1, nq * (dn + R)), bf(g, n + 1, L + R)
    slot, pos = i32([0] * (n + 1)), torch.arange(n + 1, device=DEV, dtype=torch.int32)
    put = lambda a, b, **kw: ops.mla_prep(q[a:b], kva[a:b], w, w_uk, inv_freq(), slot[a:b], pos[a:b], table, cache, page, nq, dn, L, R, 1e-6, kv_bits=bits, **kw)
    tail = put(0, n, absorb=False)
    got = ops.mla_attention_prefill(q[:n], tail, cache, kv_b, [(0, 0, n)], i32([0]), i32([n]), i32([0]), table, page, nq, dn, dv, L, R, kv_bits=bits,
                                    seg_slot=i32([0]))
    one = put(n, n + 1)
    ol = ops.mla_attention(one, cache, slot[n:], pos[n:] + 1, table, page, nq, L, R, (dn + R) ** -0.5, segs=segments(1, 1), kv_bits=bits)
    last = ops.mla_out(ol, w_uv)
    at = table[0, pos.long() // page].long() * page + pos % page
    keys = lr.unpack(cache.view(-1, cache.shape[-1])[at], L, bits).to(DEV)
    qr = q.double().view(n + 1, nq, dn + R)
    full = torch.cat([torch.einsum("thd,hld->thl", qr[..., :dn], w_uk.double()), lr.rotated(qr[..., dn:], pos, inv_freq())], -1)
    want = torch.stack([lr.attend(full[r], keys[:r + 1], L, (dn + R) ** -0.5) for r in range(n + 1)])
    want = torch.einsum("thl,hvl->thv", want, w_uv.double()).reshape(n + 1, -1)
    # keys, values, weights and results in bf16 along the way, each 2^-9 off on average: an ordinary step's rounding, as in the 16-bit cache's tests
    for a, b in ((got, want[:n]), (last, want[n:])):
        assert (a.double() - b).norm() < 8 * 2 ** -9 * b.norm()
    assert ops.status() == 0


@pytest.mark.parametrize("bits", [4, 8])
def test_captured_steps_follow_their_contexts(ops, bits):
    """A captured call replayed behind longer and shorter contexts gives what an eager call gives."""
    g = gen("graph", bits)
    L, nq, page = 512, 16, 64
    table, pages = tables([3000, 3000], page, g)
    cache = random_cache(bits, L, pages, page, g)
    q, kvlen = bf(g, 2, nq, L + R), i32([5, 7])
    call = lambda: ops.mla_attention(q, cache, i32_slots, kvlen, table, page, nq, L, R, 0.05, segs=segs, kv_bits=bits)
    i32_slots, segs = i32([0, 1]), segments(1, 2)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for lens in ([5, 7], [3000, 1], [128, 2999], [1000, 1000], [0, 64]):
        kvlen.copy_(i32(lens))
        graph.replay()
        assert torch.equal(out, call())


@pytest.mark.parametrize("bits", [4, 8])
def test_two_streams_at_once(ops, bits):
    g = gen("streams", bits)
    L, nq, page = 512, 128, 64
    table, pages = tables([2000, 1500], page, g)
    cache = random_cache(bits, L, pages, page, g)
    qs = [bf(g, 1, nq, L + R) for _ in range(2)]
    call = lambda i: ops.mla_attention(qs[i], cache, i32([i]), i32([[2000, 1500][i]]), table, page, nq, L, R, 0.05, kv_bits=bits)
    want = [call(0), call(1)]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(side[i]):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


@pytest.mark.parametrize("kv", ["int4", "fp8"])
def test_engine_over_quantised_latents(ext, kv):
    """The tiny MLA + MoE model: a prompt chunk on the expanded path, one on the absorbed rows, decode steps (captured), against the CPU engine over the
    same format; a parked and forked slot goes on as the original does."""
    from ferrite_b200.config import EngineConfig, tiny_mla
    from ferrite_b200.engine.engine import Engine
    from ferrite_b200.engine.executor import Segment
    from ferrite_b200.models.weights import init_weights
    cfg = tiny_mla()
    w = init_weights(cfg, seed=0)
    p = torch.randint(0, cfg.vocab, (110,), generator=torch.Generator().manual_seed(2)).tolist()
    ref = Engine(cfg, w, EngineConfig(n_slots=1, max_ctx=128, kv_dtype=kv), device="cpu")
    want, _, _ = ref.forward([Segment(0, 0, p, "all")])
    eng = Engine(cfg, w, EngineConfig(n_slots=2, max_ctx=128, kv_dtype=kv), device=DEV)
    assert eng.ex.k_cache[0].dtype == torch.uint8 and eng.ex.k_cache[0].shape[-1] == lr.row_bytes(64, mla_cache.BITS[kv])
    a = eng.forward([Segment(0, 0, p[:70], "all")])[0].clone()
    b = eng.forward([Segment(0, 70, p[70:100], "all")])[0].clone()
    eng.ex.copy_slot(0, 1, 100)
    tail = [eng.forward([Segment(0, 100 + i, [p[100 + i]], "last")])[0].clone() for i in range(10)]
    fork = [eng.forward([Segment(1, 100 + i, [p[100 + i]], "last")])[0].clone() for i in range(10)]
    assert all(torch.equal(x, y) for x, y in zip(tail, fork))
    got = torch.cat([a, b] + tail).float().cpu()
    kl = torch.nn.functional.kl_div(torch.log_softmax(got, -1), torch.log_softmax(want, -1), log_target=True, reduction="batchmean").item()
    assert kl < (8e-2 if kv == "int4" else 3e-2), kl             # bf16 activations, and codes that fall on the other side of a border for them
    eng.check()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nq", [128, 24])
def test_attention_in_wide_tables(ops, bits, nq, monkeypatch):
    """Tables with room for far more keys than there are: units of 64 and 32 pairs, where narrow tables have units of 16."""
    monkeypatch.setattr(sys.modules[__name__], "tables", functools.partial(tables, width=300))
    for L in (512, 256, 128, 64):
        for lens, rows, page in (((1, 127, 128, 129, 64), 1, 64), ((1000, 300), 5, 64)):
            test_attention(ops, bits, L, nq, lens, rows, page)
    test_attention_with_scores_that_grow(ops, bits, nq)
    test_values_that_are_no_numbers_reach_who_sees_them(ops, bits, nq)
    test_attention_of_rows_that_see_nothing(ops, bits)
    test_attention_scales_of_queries(ops, bits)


@pytest.mark.parametrize("width", [0, 100])
def test_attention_of_many_segments(ops, width):
    """More segments than a warp has lanes, some without rows, some that see nothing."""
    g = gen("many", width)
    n, L, nq = 71, 512, 16
    lens = [(i * 37) % 200 for i in range(n)]
    nrows = [0 if i % 9 == 4 else 1 + i % 3 for i in range(n)]
    table, pages = tables(lens, 64, g, width=width)
    cache = random_cache(4, L, pages, 64, g)
    slot = [s for s in range(n) for _ in range(nrows[s])]
    kvlen = [max(0, lens[s] - nrows[s] + 1 + r) for s in range(n) for r in range(nrows[s])]
    row0 = [sum(nrows[:s]) for s in range(n)]
    check_attention(ops, 4, L, nq, 64, slot, kvlen, table, cache, bf(g, len(slot), nq, L + R), 0.05, (i32(list(range(n))), i32(row0), i32(nrows), 3))
    seg = i32(list(range(n))), i32([max(0, lens[s] - nrows[s]) for s in range(n)]), i32([min(lens[s], nrows[s]) for s in range(n)])
    vals = lr.unpack(cache.view(-1, cache.shape[-1]), L, 4)
    total = sum(min(a, b) for a, b in zip(lens, nrows))
    got = ops.mla_rows(cache, *seg, table, 64, L, R, total, kv_bits=4).cpu().double()
    want = [int(table[s, p // 64]) * 64 + p % 64 for s in range(n) for p in range(max(0, lens[s] - nrows[s]), lens[s])]
    assert torch.equal(got, vals[want])
    got = ops.mla_rows(cache, *seg, table, 64, L, R, sum((m + 63) // 64 * 64 for m in lens), whole=True, kv_bits=4).cpu().double()
    lo = 0
    for s, m in enumerate(lens):
        assert torch.equal(got[lo:lo + m], vals[[int(table[s, p // 64]) * 64 + p % 64 for p in range(m)]])
        lo += (m + 63) // 64 * 64


@pytest.mark.parametrize("bits", [4, 8])
def test_prep_reads_rows_on_any_address(ops, bits):
    g = gen("address", bits)
    T, L = 9, 512
    table, pages = tables([T], 64, g)
    wide = bf(g, T, L + R + 5)
    slot, pos = [0] * T, list(range(T))
    _, odd, before, q, kva, w = prep(ops, bits, L, 2, 16, slot, pos, table, pages, 64, g, kva=wide[:, 3:3 + L + R])
    even = before.clone()
    ops.mla_prep(q, kva.contiguous(), w, None, inv_freq(), i32(slot), i32(pos), table, even, 64, 2, 16, L, R, 1e-6, absorb=False, kv_bits=bits)
    assert torch.equal(odd, even) and not torch.equal(odd, before)


@pytest.mark.parametrize("width", [0, 300])
@pytest.mark.parametrize("falling", [False, True])
def test_attention_with_scores_past_what_32_bits_tell_apart(ops, width, falling):
    """Scores of 4e9 a step, rising or falling along the keys: all weight is one key's, whose value comes back, off by its rounding to bf16 and
    by that of its weight (2^-8 and 2^-11)."""
    g = gen("huge", width)
    n, L, nq = 256, 512, 128
    table, pages = tables([n], 64, g, width=width)
    cache = random_cache(4, L, pages, 64, g)
    p = torch.arange(n, device=DEV)
    flat = table[0, p // 64].long() * 64 + p % 64
    rope = torch.zeros(n, R, dtype=torch.bfloat16, device=DEV)
    rope[:, 0] = n - 1 - p if falling else p
    cache.view(-1, cache.shape[-1])[flat, L // 2:L // 2 + 2 * R] = rope.view(torch.uint8).view(n, 2 * R)
    q = torch.zeros(1, nq, L + R, dtype=torch.bfloat16, device=DEV)
    q[..., L] = 2.0 ** 36
    got = ops.mla_attention(q, cache, i32([0]), i32([n]), table, 64, nq, L, R, 1 / 16, segs=segments(1, 1), kv_bits=4)
    want = lr.unpack(cache.view(-1, cache.shape[-1])[flat[0 if falling else -1]][None], L, 4)[:, :L].to(DEV)
    assert ((got[0].double() - want).abs() <= want.abs() * (2 ** -8 + 2 ** -11)).all()
