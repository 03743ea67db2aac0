"""Ops over a page pool that streams share, on the GPU, where inputs are out of the ordinary: values and keys that are no finite numbers, tables that leave
out what is read through others, pages that come twice, tables wider than the contexts, calls of everything captured and replayed."""
import zlib

import pytest
import shared_pages
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF, NAN = float("inf"), float("nan")
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


def attend(ops, st, **kw):
    return ops.attention_shared(st.q, None, st.k, st.v, st.kvlen, *st.args(), False, st.segs, st.groups, want_lse=True, **kw)


def sums(ops, st, lse=None, carry=0.5, **kw):
    return ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups, lse=lse, carry=carry, out=st.mass.clone(), **kw)


def alike(got, want, tol):
    """Infinities and NaN in the same places, everything else within `tol`."""
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got.double()[inf], want[inf])
    off = (got.double() - want).abs()
    assert (off <= tol)[fin].all(), float((off / tol)[fin].max())


def check_attend(st, out, lse):
    want, wl, tol, ltol = st.attend()
    # rounded to bf16 once: half a step, 2^-8 of the value that is rounded
    alike(out.view_as(want), want, tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30)
    alike(lse, wl, ltol)


def check_sums(st, got, carry, lse=None):
    want, tol, seen = st.masses(carry, lse)
    assert torch.equal(got[~seen], st.mass[~seen])
    alike(got, want, tol)


# ---- values and keys that are no finite numbers ------------------------------------------------------------------------

def stream_row(st, s, token):
    """Row of the caches where a token of stream s lies."""
    gi = st.member[s]
    via = st.first[gi] if gi is not None and token < st.shared[gi] else s
    return int(st.table[st.slots[via], token // st.page]) * st.page + token % st.page


@pytest.mark.parametrize("nq,nkv,hd", [(6, 2, 128), (24, 4, 256), (4, 2, 64)])
def test_values_that_are_no_finite_numbers(ops, nq, nkv, hd):
    """Such a value shows in its own column of the rows that see it, an infinity as itself; the logarithms and the sums made with them know nothing of values.
    In tiles that all rows see, that some see, that the shared tokens end in, of a stream's own."""
    def step():
        return shared_pages.Step(gen("values", nq, hd), DEV, nq, nkv, hd, 64, ((200, [[230, 210, 226], [260]]), (3000, [[3100, 3060]])), [[40, 30, 35], [700]])
    st = step()
    places = [(0, 220, 0, 5, INF), (0, 221, 0, 8, INF), (0, 222, 0, 8, -INF), (0, 223, 1, 7, NAN), (0, 10, 0, 9, -INF), (0, 198, 1, 20, INF), (1, 259, 1, 33, -INF),
              (2, 100, 0, 1, INF), (2, 2999, 0, 2, -INF), (2, 3080, 1, hd - 1, INF), (3, 33, 0, 0, INF), (3, 3, 0, 63, INF), (3, 4, 0, 63, NAN), (4, 500, 1, 11, -INF),
              (4, 699, 1, 12, INF)]
    for s, token, head, column, value in places:
        st.v.view(-1, nkv, hd)[stream_row(st, s, token), head, column] = value
    out, lse = attend(ops, st)
    check_attend(st, out, lse)
    plain, plain_lse = attend(ops, step())
    assert torch.equal(lse, plain_lse)
    fin = torch.isfinite(out)
    assert torch.equal(out[fin], plain[fin])
    check_sums(st, sums(ops, st, lse), 0.5)


def test_rows_whose_values_are_all_infinite(ops):
    """Every value of a head infinite, of one sign and of both; gated too."""
    st = shared_pages.Step(gen("all infinite"), DEV, 6, 2, 128, 64, ((130, [[140, 131], [200]]),), [[9, 3]])
    st.v[:, :, 0, :40] = INF
    st.v[:, :, 0, 40:60] = -INF
    st.v[:, ::2, 0, 60:] = INF
    st.v[:, 1::2, 0, 60:] = -INF
    check_attend(st, *attend(ops, st))
    proj = torch.randn(st.rows, 6 * 256, generator=gen("gate"), device=DEV).to(torch.bfloat16)
    got = ops.attention_shared(st.q, proj, st.k, st.v, st.kvlen, *st.args(), True, st.segs, st.groups)
    assert torch.equal(got.view(-1, 6, 128)[:, :3].float().nan_to_num(7, 8, 9), attend(ops, st)[0].view(-1, 6, 128)[:, :3].float().nan_to_num(7, 8, 9))


class OddKeys(shared_pages.Step):
    """A step with keys that are no finite numbers: rounding leaves what it leaves of the scores of the others."""

    def weights(self, t):
        x, l, _ = super().weights(t)
        k = self.k.reshape(-1, self.nkv, self.hd)[self.at(t)].double().nan_to_num(0, 0, 0)
        off = (torch.einsum("kgd,tkd->kgt", self.q[t].reshape(self.nkv, -1, self.hd).double().abs(), k.abs()) / self.hd ** 0.5).amax(-1) * 2.0 ** -20
        return x, l, off

    def check_sums(self, got, carry, lse=None):
        want, tol, seen = self.masses(carry, lse)
        assert torch.equal(got[~seen], self.mass[~seen])
        alike(got, want, torch.where(torch.isnan(tol), 2.0 ** -22 * want.abs(), tol))       # (where a score is minus infinity for every row: nothing is added)


def odd_keys(nq, nkv, hd):
    """Heads that look at column 0 all the same way, and keys with infinities there: scores of infinity, minus infinity, NaN."""
    st = OddKeys(gen("scores", nq, hd), DEV, nq, nkv, hd, 64, ((200, [[230, 210, 226], [260]]), (3000, [[3100, 3060]])), [[40, 30, 35], [700]])
    st.q[:, :, 0] = st.q[:, :, 0].abs() + 0.1
    flat = st.k.view(-1, nkv, hd)
    for s, token, head, value in [(0, 220, 0, INF), (1, 255, 1, -INF), (2, 100, 0, INF), (2, 2990, 1, -INF), (2, 3090, 1, NAN), (3, 33, 1, INF), (3, 31, 1, NAN),
                                  (4, 650, 0, -INF), (4, 65, 1, INF)]:
        flat[stream_row(st, s, token), head, 0] = value
    return st


@pytest.mark.parametrize("nq,nkv,hd", [(6, 2, 128), (24, 4, 256), (4, 2, 64)])
def test_scores_of_infinity(ops, nq, nkv, hd):
    """A score of infinity makes the logarithm infinity, NaN only where another score of the row is NaN; the row's output is NaN. Scores of minus infinity weigh nothing."""
    st = odd_keys(nq, nkv, hd)
    wl = st.attend()[1]
    assert torch.isposinf(wl).any() and torch.isnan(wl).any() and torch.isfinite(wl).any()
    check_attend(st, *attend(ops, st))


def test_sums_of_scores_of_infinity(ops):
    st = odd_keys(4, 2, 64)
    for lse in (None, attend(ops, st)[1]):
        st.check_sums(sums(ops, st, lse), 0.5)


# ---- tables ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("nq,nkv,hd", [(6, 2, 128), (24, 4, 256), (4, 2, 64)])
@pytest.mark.parametrize("shared", [64, 192, 320, 321])
@pytest.mark.parametrize("rows", [1, 300])
def test_streams_need_no_entries_for_shared_pages(ops, nq, nkv, hd, shared, rows):
    """Shared tokens are read through the table of a group's first stream: whole pages of them are missing from the others' tables."""
    members = [[shared + 5], [max(0, shared + 100 - i) for i in range(rows)], [shared + 1]]
    st = shared_pages.Step(gen("no entries", nq, shared, rows), DEV, nq, nkv, hd, 64, ((shared, members),), [[70]])
    full = st.table.clone()
    st.table[st.slots[1]:st.slots[2] + 1, :shared // 64] = -1
    out, lse = attend(ops, st)
    got = [sums(ops, st), sums(ops, st, lse)]
    assert ops.status() == 0
    st.table.copy_(full)                                                 # (the statement in 64 bits is the same for both)
    check_attend(st, out, lse)
    for g in got:
        check_sums(st, g, 0.5)


@pytest.mark.parametrize("nq,nkv,hd", [(24, 4, 256), (6, 2, 128), (5, 1, 128), (11, 1, 64), (33, 1, 64), (4, 2, 64)])
@pytest.mark.parametrize("rows", [8, 24, 300])
def test_sums_beside_keys_of_minus_infinity(ops, nq, nkv, hd, rows):
    """A key whose score is minus infinity for every row gets nothing, also where the query heads of whole rows leave some of a product's columns without a pair."""
    st = OddKeys(gen("minus", nq, hd, rows), DEV, nq, nkv, hd, 64, alone=[[700 - r for r in range(rows)]])
    st.q[:, :, 0] = st.q[:, :, 0].abs() + 0.1
    for token in (0, 50, 127, 200, 399):
        st.k.view(-1, nkv, hd)[stream_row(st, 0, token), :, 0] = -INF
    for lse in (None, attend(ops, st)[1]):
        got = sums(ops, st, lse)
        assert torch.isfinite(got).all()
        st.check_sums(got, 0.5)


# ---- eviction ----------------------------------------------------------------------------------------------------------

def pool(g, lens, keep, page, nkv, row, width=0, levels=0):
    """A pool of bf16 rows with streams of `lens` tokens in tables of `width` entries, or as many as the longest has; sums of few levels where said."""
    need, per = [-(-n // page) for n in lens], -(-keep // page)
    total = sum(need) + len(lens) * per + 1
    order = torch.randperm(total, generator=g, device=DEV).int()
    table, at = torch.full((len(lens), max(need + [width])), -1, dtype=torch.int32, device=DEV), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    dst = order[at:at + len(lens) * per].view(len(lens), per).contiguous()
    k, v = (torch.randn(total, page, nkv, row, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    mass = (torch.randint(0, levels, (total, nkv, page), generator=g, device=DEV).float() if levels else torch.randn(total, nkv, page, generator=g, device=DEV).exp())
    return table, dst, k, v, mass


def check_evict(ops, lens, keep, first, recent, page, nkv, table, dst, k, v, mass):
    """Against a sort of every context, whole pools compared."""
    old = [x.clone() for x in (k, v, mass)]
    kept = ops.kv_evict(k, v, None, mass, i32(list(range(len(lens)))), i32(lens), table, dst, page, keep, first, recent)
    want = [x.clone() for x in old]
    for s, n in enumerate(lens):
        pos, i = torch.arange(n, device=DEV), torch.arange(min(n, keep), device=DEV)
        w = old[2].transpose(1, 2)[table[s, pos // page].long(), pos % page]                     # [tokens, heads]
        for h in range(nkv):
            ids = pos
            if n > keep:
                best = torch.sort(w[first:n - recent, h], descending=True, stable=True).indices[:keep - first - recent] + first
                ids = torch.cat([pos[:first], best.sort().values, pos[n - recent:]])
            assert torch.equal(kept[s, h], torch.cat([ids.int(), i32([-1] * (keep - len(ids)))]))
            a, b, c, d = table[s].long()[ids // page], ids % page, dst[s].long()[i // page], i % page
            for x, was in zip(want[:2], old[:2]):
                x[c, d, h] = was[a, b, h]
            want[2][c, h, d] = old[2][a, h, b]
    for x, y in zip((k, v, mass), want):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("streams,nkv", [(1, 1), (1, 4), (5, 4), (24, 4), (40, 4)])
@pytest.mark.parametrize("width", [70, 300, 2048, 20000])
def test_evict_with_wide_tables(ops, streams, nkv, width):
    """Tables with room for far more than the contexts: the same tokens, however many CTAs the room asks for."""
    lens = [1 + (1237 * i + 4000) % 4400 for i in range(streams)]
    for levels in (0, 3):
        check_evict(ops, lens, 500, 3, 101, 64, nkv, *pool(gen("wide", streams, width, levels), lens, 500, 64, nkv, 8, width, levels))


@pytest.mark.parametrize("streams,nkv,longest,levels", [(1, 1, 200000, 0), (1, 1, 200000, 4), (1, 1, 400000, 0), (1, 1, 400000, 4), (19, 4, 50000, 0), (19, 4, 50000, 3),
                                                        (38, 4, 22000, 4)])
def test_evict_of_very_long_contexts(ops, streams, nkv, longest, levels):
    """More tokens a CTA than a warp keeps track of in registers, and more than shared memory holds the weights of; equal ones across all of it."""
    lens = [max(1, longest - 997 * i) for i in range(streams)]
    check_evict(ops, lens, 3001, 5, 700, 64, nkv, *pool(gen("very long", streams, longest, levels), lens, 3001, 64, nkv, 8, 0, levels))


# ---- keys of two segments ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("spoil", ["forked twice", "forked in a page", "slot", "page", "group"])
def test_sums_of_keys_that_two_segments_hold(ops, rows, spoil):
    """A key's sum is written once: one that two segments hold, or a segment and a group's shared tokens, is reported. The attention takes such steps."""
    def some(n):
        return [max(1, n - i) for i in range(rows)]

    def step():
        return shared_pages.Step(gen("forked", rows), DEV, 6, 2, 128, 64, ((128, [[130], some(900), [1000]]),), [[333], [64]], poison=None)
    st = step()
    attend(ops, st)
    check_sums(st, sums(ops, st), 0.5)                                   # nothing held twice, nothing reported
    assert ops.status() == 0
    if spoil == "forked twice":
        st.table[2, 2:13] = st.table[1, 2:13]
    elif spoil == "forked in a page":
        st.table[2, 14] = st.table[1, 14]                                # token 896 .. 899 of one, 896 .. 959 of the other
    elif spoil == "slot":
        st.segs[0][3] = 2
    elif spoil == "page":
        st.table[3, 5] = st.table[3, 2]                                  # its last page again, ahead of the last tokens
    else:
        st.table[4, 0] = st.table[0, 1]                                  # a shared page as another stream's own
    lse = attend(ops, st)[1]
    assert ops.status() == 0
    for known in (lse, None):
        sums(ops, st, known)
        assert ops.status() != 0
        ops.status_word.zero_()


# ---- empty calls -------------------------------------------------------------------------------------------------------

def test_calls_without_rows_or_segments(ops):
    """Steps of no rows and of no segments launch nothing, count nothing and leave everything as it was."""
    st = shared_pages.Step(gen("empty"), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[9]])
    table, dst, k, v, mass = pool(gen("empty evict"), [100], 32, 64, 2, 8)
    none = i32([])
    before, launches = [x.clone() for x in (st.mass, k, v, mass)], ops.launches
    for q, kvlen, segs in ((st.q[:0], none, st.segs), (st.q, st.kvlen, (none, none, none, 0)), (st.q[:0], none, (none, none, none, 0))):
        out, lse = ops.attention_shared(q, None, st.k, st.v, kvlen, *st.args(), False, segs, want_lse=True)
        assert out.shape == (len(q), 768) and lse.shape == (len(q), 6)
        for known in (None, lse):
            ops.attention_mass(q, st.k, st.mass, kvlen, *st.args(), segs, lse=known)
    assert ops.kv_evict(k, v, None, mass, none, none, table, dst[:0], 64, 32).shape == (0, 2, 32)
    assert ops.launches == launches
    for x, y in zip((st.mass, k, v, mass), before):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---- layouts ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [3, 300])
def test_one_query_for_all_rows(ops, rows):
    """A query expanded over the rows, and rows that overlap: the same as a copy of them."""
    st = shared_pages.Step(gen("expanded", rows), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[500 - i for i in range(rows - 2)]])
    flat = torch.randn(6 * 128 + 8 * rows, generator=gen("overlap"), device=DEV).to(torch.bfloat16)
    for q in (st.q[:1].expand(rows, 6, 128), flat.as_strided((rows, 6, 128), (8, 128, 1))):
        st.q = q
        got = [attend(ops, st), sums(ops, st)]
        st.q = q.contiguous()
        want = [attend(ops, st), sums(ops, st)]
        assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[0][1], want[0][1]) and torch.equal(got[1], want[1])
        check_sums(st, got[1], 0.5)


# ---- steps of very many rows -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("nq,hd", [(1, 64), (3, 128)])
def test_steps_whose_lengths_do_not_fit_beside_the_plan(ops, nq, hd):
    """More rows than the plan has room for the lengths of: they are read where they lie."""
    rows, n, page = 41500, 300, 64
    g = gen("rows", nq)
    k, v = (torch.randn(8, page, 1, hd, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    table = torch.randperm(8, generator=g, device=DEV).int()[:5].view(1, 5).contiguous()
    q = torch.randn(rows, nq, hd, generator=g, device=DEV).to(torch.bfloat16)
    kvlen = torch.randint(0, n + 1, (rows,), generator=g, device=DEV, dtype=torch.int32)
    segs = (i32([0]), i32([0]), i32([rows]), rows)
    out, lse = ops.attention_shared(q, None, k, v, kvlen, table, page, nq, 1, hd, False, segs, want_lse=True)
    at = table[0].long()[torch.arange(n, device=DEV) // page] * page + torch.arange(n, device=DEV) % page
    keys, values = k.view(-1, hd)[at].double(), v.view(-1, hd)[at].double()
    sees = torch.arange(n, device=DEV) < kvlen[:, None, None]
    x = torch.where(sees, q.double() @ keys.t() / hd ** 0.5, -INF)
    wl = torch.logsumexp(x, -1)
    p = torch.where(sees, torch.exp(x - wl[..., None]), 0.0)
    # as in shared_pages.Step: scores in 32 bits, weights of twice eight bits
    off = torch.where(sees, q.double().abs() @ keys.abs().t(), 0.0).amax(-1) / hd ** 0.5 * 2.0 ** -20
    tol = (p @ values.abs()) * (2 * (off[..., None] + 2.0 ** -20) + 2.0 ** -16 + 2.0 ** -12)
    want = p @ values
    alike(out.view_as(want), want, tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30)
    alike(lse, wl, off + 2.0 ** -22 * wl.abs().nan_to_num(0, 0, 0) + 2.0 ** -20)
    rel = off[..., None] * 2 + 2.0 ** -20 + 2.0 ** -22 * (x.abs().nan_to_num(0, 0, 0) + wl.abs().nan_to_num(0, 0, 0)[..., None])
    new, mtol = p.sum((0, 1)), (p * rel).sum((0, 1))
    mtol += new * (rows * nq) * 2.0 ** -24 + 2.0 ** -22 * new
    for known in (lse, None):
        got = ops.attention_mass(q, k, torch.zeros(8, 1, page, device=DEV), kvlen, table, page, nq, 1, hd, segs, lse=known)
        alike(got.view(-1)[at], new, mtol)
        assert float(got.sum()) == float(got.view(-1)[at].sum())


def test_steps_of_more_rows_than_a_call_plans(ops):
    """Refused, with what the bound is for."""
    rows = 20600
    q = torch.zeros(rows, 128, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(2, 64, 1, 64, dtype=torch.bfloat16, device=DEV)
    kvlen, table, segs = i32([10] * rows), i32([[0, 1]]), (i32([0]), i32([0]), i32([rows]), rows)
    with pytest.raises(RuntimeError, match="more segments or rows than a call plans"):
        ops.attention_shared(q, None, k, k, kvlen, table, 64, 128, 1, 64, False, segs)
    with pytest.raises(RuntimeError, match="more segments or rows than a call plans"):
        ops.attention_mass(q[:, :64], k, torch.zeros(2, 1, 64, device=DEV), kvlen, table, 64, 64, 1, 64, segs, lse=torch.zeros(rows, 64, device=DEV))


# ---- steps that are wrong in a part ------------------------------------------------------------------------------------

@pytest.mark.parametrize("fill", [0x7fffffff, -1, 1 << 20])
@pytest.mark.parametrize("spoil", ["rows", "slot"])
@pytest.mark.parametrize("many", [False, True])
def test_sums_beside_refused_segments(ops, fill, spoil, many):
    """A segment that does not fit the step sets the status. The sums of the others' keys are right, whatever the workspace held, and nothing else changes."""
    rows = 150 if many else 3
    st = shared_pages.Step(gen("refused sums", spoil, many), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[9], [31 + i for i in range(rows)], [77]], spare=20)
    bad = 3
    if spoil == "rows":
        segs = (*st.segs[:3], rows - 1)
    else:
        segs = (i32([*st.segs[0][:bad].tolist(), -5, int(st.segs[0][4])]), *st.segs[1:])
    lse = attend(ops, st)[1]
    ops.status_word.zero_()
    want, tol, seen = st.masses(0.5)
    other = torch.ones(st.k.shape[0], dtype=torch.bool, device=DEV)      # pages of the other streams and of none
    other[st.table[st.slots[bad]][st.table[st.slots[bad]] >= 0].long()] = False
    for known in (lse, None):
        n = ops.C.attention_mass_floats(st.rows, 5, segs[3], 1, 6, 2, 128, st.table.shape[1] * 64, st.k.shape[0] * 64, known is None, ops.sm_count)
        out = st.mass.clone()
        torch.full((n,), fill, dtype=torch.int32, device=DEV)            # what the allocator hands out next
        ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), segs, st.groups, lse=known, carry=0.5, out=out)
        assert ops.status() != 0
        ops.status_word.zero_()
        assert ((out - want).abs() <= tol)[seen & other[:, None, None]].all()
        assert torch.equal(out[~seen], st.mass[~seen]) and torch.equal(out[~other], st.mass[~other])


def test_wrong_tables_touch_nothing_else(ops):
    """Pages that are none, contexts beyond the table, slots that are none: caches, tables and sums that the step does not name stay as they were."""
    for spoil in ("page", "far page", "length", "slot", "group"):
        st = shared_pages.Step(gen("wrong", spoil), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[9]], spare=30, poison=None)
        named = torch.zeros(st.k.shape[0], dtype=torch.bool, device=DEV)
        named[st.table[st.table >= 0].long()] = True
        if spoil == "page":
            st.table[0, 1] = -1
        elif spoil == "far page":
            st.table[1, 3] = 1 << 30
        elif spoil == "length":
            st.kvlen[2] = 100000
        elif spoil == "slot":
            st.segs[0][2] = 77
        else:
            st.groups[0][0] = 3
        held = [t.clone() for t in (st.k, st.v, st.mass, st.table, st.kvlen, st.q)]
        lse = attend(ops, st)[1]
        outs = [sums(ops, st, known) for known in (lse, None)]
        assert ops.status() != 0, spoil
        ops.status_word.zero_()
        for t, h in zip((st.k, st.v, st.mass, st.table, st.kvlen, st.q), held):
            assert torch.equal(t, h), spoil
        for out in outs:
            assert torch.equal(out[~named], st.mass[~named]), spoil
    for spoil in ("page", "dst", "length", "slot"):
        table, dst, k, v, mass = pool(gen("wrong evict", spoil), [200, 150], 64, 64, 2, 8)
        new = torch.zeros(k.shape[0], dtype=torch.bool, device=DEV)
        new[dst.long()] = True
        n, slot = i32([200, 150]), i32([0, 1])
        if spoil == "page":
            table[0, 2] = 1 << 20
        elif spoil == "dst":
            new[dst[0, 0].long()] = False
            dst[0, 0] = -1
        elif spoil == "length":
            n[0] = 1 << 20
        else:
            slot[0] = -1
        held = [t.clone() for t in (k, v, mass)]
        ops.kv_evict(k, v, None, mass, slot, n, table, dst, 64, 64, 2, 10)
        assert ops.status() != 0, spoil
        ops.status_word.zero_()
        for t, h in zip((k, v, mass), held):
            assert torch.equal(t[~new], h[~new]), spoil


# ---- captured calls ----------------------------------------------------------------------------------------------------

def captured(call):
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = call()
    return graph, res


def test_captured_sums_follow_their_tables(ops):
    """Attention, the sums of a step's few rows and those of a prompt, their logarithms in hand and not, each captured and replayed with other pages, lengths and queries."""
    few = lambda seed, lens: shared_pages.Step(gen("captured few", seed), DEV, 8, 2, 128, 64, ((256, [[lens[0]], [lens[1]], [lens[2]]]),), [[lens[3]]], poison=None, spare=12,
                                               width=4)
    many = lambda seed, lens: shared_pages.Step(gen("captured many", seed), DEV, 24, 4, 256, 64, (), [list(range(n - r + 1, n + 1)) for n, r in zip(lens, (200, 70))],
                                                poison=None, spare=14, width=4)
    for make, lens, more in ((few, (400, 310, 555, 70), ((290, 600, 257, 1), (256, 480, 301, 190))), (many, (700, 300), ((200, 640), (650, 90)))):
        st = make(0, lens)
        st.mass.fill_(1.0)
        out = torch.zeros_like(st.mass)

        def call():
            o, lse = attend(ops, st)
            ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups, lse=lse, carry=0.5, out=out)
            alone = ops.attention_mass(st.q, st.k, torch.zeros_like(st.mass), st.kvlen, *st.args(), st.segs, st.groups, carry=0.0)
            return o, lse, alone
        graphs = [captured(call) for _ in range(2)]
        for i, now in enumerate((lens, *more)):
            if i:
                nxt = make(i, now)
                pages = min(st.k.shape[0], nxt.k.shape[0])
                width = min(st.table.shape[1], nxt.table.shape[1])
                assert int(nxt.table.max()) < st.k.shape[0] and (nxt.table[:, width:] < 0).all()
                st.k[:pages], st.v[:pages] = nxt.k[:pages], nxt.v[:pages]
                st.q.copy_(nxt.q); st.kvlen.copy_(nxt.kvlen)
                st.table.fill_(-1)
                st.table[:, :width] = nxt.table[:, :width]
                st.streams = nxt.streams
            want, tol, seen = st.masses(0.5)
            zero, ztol, _ = st.masses(0.0)
            for graph, (o, lse, alone) in graphs:
                out.fill_(7.0)
                graph.replay()
                torch.cuda.synchronize()
                check_attend(st, o, lse)
                assert ((out - want).abs() <= tol)[seen].all() and (out[~seen] == 7).all()
                assert ((alone - zero).abs() <= ztol)[seen].all() and (alone[~seen] == 0).all()


def test_captured_eviction_follows_its_tables(ops):
    """A captured eviction replayed with other lengths, pages and sums, in a table wider than any context."""
    keep, page, nkv = 300, 64, 2
    first = pool(gen("captured evict", 0), [299, 301, 10000], keep, page, nkv, 8, 400)
    table, dst, k, v, mass = (t.clone() for t in first)
    lens, slots = i32([299, 301, 10000]), i32([0, 1, 2])
    graph, kept = captured(lambda: ops.kv_evict(k, v, None, mass, slots, lens, table, dst, page, keep, 4, 50))
    for i, now in enumerate(([299, 301, 10000], [8000, 1200, 1], [1000, 300, 9000], [0, 5000, 4000])):
        nt, nd, nk, nv, nm = pool(gen("captured evict", i), now, keep, page, nkv, 8, 400)
        n = nk.shape[0]
        assert n <= k.shape[0] and nt.shape == table.shape
        table.copy_(nt); dst.copy_(nd); lens.copy_(i32(now))
        for t, x in zip((k, v, mass), (nk, nv, nm)):
            t[:n] = x
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.kv_evict(nk, nv, None, nm, slots, i32(now), nt, nd, page, keep, 4, 50)
        assert torch.equal(kept, eager)
        for t, x in zip((k, v, mass), (nk, nv, nm)):
            assert torch.equal(t[:n].view(torch.uint8), x.view(torch.uint8))
        check_evict(ops, now, keep, 4, 50, page, nkv, *pool(gen("captured evict", i), now, keep, page, nkv, 8, 400))


def test_contexts_that_were_shrunk(ops):
    """Sums of a step, eviction by them, attention over what stayed, to the precision of weights of twice eight bits; then a token is appended, whose sum its writer clears."""
    nq, nkv, hd, page, keep = 8, 2, 128, 64, 200
    st = shared_pages.Step(gen("shrunk"), DEV, nq, nkv, hd, page, ((640, [[900], [700], [1000]]),), [[333]], spare=4 * 4 + 2, poison=None, q_scale=2.0)
    mass = torch.full_like(st.mass, 5.0)                                 # what former owners left
    out, lse = attend(ops, st)
    ops.attention_mass(st.q, st.k, mass, st.kvlen, *st.args(), st.segs, st.groups, lse=lse, carry=0.0)
    used = torch.zeros(st.k.shape[0], dtype=torch.bool, device=DEV)
    used[st.table[st.table >= 0].long()] = True
    dst = torch.nonzero(~used).flatten()[:16].int().view(4, 4).contiguous()
    kept = ops.kv_evict(st.k, st.v, None, mass, i32(st.slots), i32([900, 700, 1000, 333]), st.table, dst, page, keep, 4, 64)
    assert (mass[dst[:, 3].long()][:, :, keep % page:] == 5).all()       # behind the last token: as it was
    new = shared_pages.Step.__new__(shared_pages.Step)
    new.__dict__.update(st.__dict__)
    new.table, new.slots, new.member, new.groups, new.first = dst, [0, 1, 2, 3], [None] * 4, None, {}
    new.segs = (i32([0, 1, 2, 3]), *st.segs[1:])
    new.streams, new.kvlen = [[keep]] * 4, i32([keep] * 4)
    check_attend(new, *attend(ops, new))
    # the next token
    page_of, place = dst[:, keep // page].long(), keep % page
    st.k[page_of, place], st.v[page_of, place] = st.q[:, :nkv], st.q[:, nkv:2 * nkv]
    mass[page_of, :, place] = 0
    new.streams, new.kvlen, new.mass = [[keep + 1]] * 4, i32([keep + 1] * 4), mass.clone()
    out, lse = attend(ops, new)
    check_attend(new, out, lse)
    check_sums(new, sums(ops, new, lse, 1.0), 1.0)
