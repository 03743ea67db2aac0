"""Ops over a page pool that streams share, on the GPU: attention over a common prefix, sums of weights and eviction against 64 bits, alone and one after
the other as a server runs them."""
import zlib

import pytest
import shared_pages
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
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


def attend(ops, st, want_lse=True, q=None, **kw):
    return ops.attention_shared(st.q if q is None else q, None, st.k, st.v, st.kvlen, *st.args(), False, st.segs, st.groups, want_lse=want_lse, **kw)


def check_attend(st, out, lse):
    want, wl, tol, ltol = st.attend()
    got = out.view_as(want).double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    # rounded to bf16 once: half a step, 2^-8 of the value (of the value that is rounded)
    assert ((got - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30)[~nan].all()
    if lse is not None:
        fin = torch.isfinite(wl)
        assert torch.equal(lse.double()[~fin].nan_to_num(7, 8, 9), wl[~fin].nan_to_num(7, 8, 9))
        assert ((lse - wl).abs() <= ltol)[fin].all()


HEADS = [(24, 4, 256), (16, 2, 256), (32, 8, 128), (3, 3, 128), (4, 2, 64), (12, 1, 64)]
# (shared tokens, own streams) .., streams of no group
STEPS = {
    "one row": ((), [[1]]),
    "one token each, two rows": ((), [[1], [1]]),
    "whole tiles": (((128, [[128 + 64], [128 + 1], [128]]),), []),
    "ends inside tiles and pages": (((201, [[230], [202], [201], [333]]), (63, [[64], [190]])), [[77], [500]]),
    "nothing shared": (((0, [[5], [70]]),), [[3]]),
    "one shared token": (((1, [[1], [2], [66]]),), []),
    "several rows a stream": (((500, [[598, 599, 600], [505], list(range(530, 547))]),), [list(range(1, 18))]),
    "rows in any order, some see nothing": (((100, [[150, 3, 0, 149], [100, 101]]), (70, [[0], [71]])), [[0], [9, 0, 8]]),
    "empty segments": (((90, [[], [95]]),), [[], [4]]),
    "more pairs than a tile": (((640, [[650 + 3 * i] for i in range(45)]),), [[900]]),
}


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("name", STEPS)
def test_attention(ops, name, nq, nkv, hd):
    groups, alone = STEPS[name]
    g = gen("attend", name, nq, hd)
    st = shared_pages.Step(g, DEV, nq, nkv, hd, {64: 64, 128: 192, 256: 128}[hd], groups, alone, width=1)
    out, lse = attend(ops, st)
    check_attend(st, out, lse)
    assert torch.equal(out, attend(ops, st, want_lse=False))


@pytest.mark.parametrize("nq,nkv,hd,streams,shared,own", [(24, 4, 256, 6, 8000, 900), (32, 8, 128, 64, 3000, 130), (4, 2, 64, 3, 20000, 5000), (24, 4, 256, 1, 0, 30000),
                                                          (5, 1, 128, 40, 700, 900)])
def test_attention_of_long_contexts(ops, nq, nkv, hd, streams, shared, own):
    g = gen("long", nq, hd, streams)
    members = [[shared + max(1, own * (i + 3) // (streams + 3))] for i in range(streams)]
    st = shared_pages.Step(g, DEV, nq, nkv, hd, 64, ((shared, members),) if shared else (), [] if shared else members, q_scale=2.0)
    check_attend(st, *attend(ops, st))


def test_scores_of_every_size(ops):
    """Scores up to hundreds, ever larger along the context (the maximum moves), all equal ones, heavy single keys."""
    for scale, ramp in ((20.0, False), (1.0, True), (0.0, False)):
        st = shared_pages.Step(gen("scores", scale), DEV, 8, 2, 128, 64, ((300, [[700], [301]]),), [[650]], q_scale=scale)
        if ramp:
            at = torch.arange(st.k.shape[0] * 64, device=DEV) % 1000
            way = torch.randn(128, generator=gen("way"), device=DEV)
            st.k.view(-1, 2, 128).copy_((st.k.view(-1, 2, 128).float() * 0.1 + at[:, None, None] * 0.01 * way).to(torch.bfloat16))
            st.q.copy_((way + 0.1 * st.q.float()).to(torch.bfloat16))
        check_attend(st, *attend(ops, st))


@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_keys_and_values_that_are_no_numbers(ops, what):
    """Rows that do not see the token stay clean, wherever it lies; those that see it have no finite result."""
    for which in ("k", "v"):
        st = shared_pages.Step(gen("bad", which), DEV, 6, 2, 128, 64, ((200, [[230, 210, 226], [260]]),), [[40, 30, 35]])
        page = st.table[st.slots[0], 220 // 64]
        getattr(st, which)[page, 220 % 64] = what                       # token 220 of the first stream: rows of 230 and 226 see it
        st2 = shared_pages.Step(gen("bad", which), DEV, 6, 2, 128, 64, ((200, [[230, 210, 226], [260]]),), [[40, 30, 35]])
        out, lse = attend(ops, st)
        clean, clean_lse = attend(ops, st2)
        sees = torch.tensor([True, False, True, False, False, False, False], device=DEV)
        assert torch.equal(out[~sees], clean[~sees]) and torch.equal(lse[~sees], clean_lse[~sees])
        if which == "v" or what != what:
            assert not torch.isfinite(out[sees].float().sum(-1)).any()


def test_layouts_of_the_queries(ops):
    st = shared_pages.Step(gen("layout"), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[9]])
    want = attend(ops, st)
    wide = torch.full((3, 6 * 128 + 40), float("nan"), dtype=torch.bfloat16, device=DEV)
    for off in (0, 8, 3):
        wide[:, off:off + 768] = st.q.view(3, -1)
        for q in (wide[:, off:off + 768], wide[:, off:off + 768].unflatten(1, (6, 128))):
            got = attend(ops, st, q=q)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    turned = st.q.transpose(0, 1).contiguous().transpose(0, 1)          # heads ahead of rows
    assert torch.equal(attend(ops, st, q=turned)[0], want[0])


def test_gate(ops):
    st = shared_pages.Step(gen("gate"), DEV, 24, 4, 256, 64, ((130, [[140], [200]]),), [[9]])
    proj = torch.randn(3, 24 * 512 + 11, generator=gen("proj"), device=DEV).to(torch.bfloat16)[:, 1:]
    out = ops.attention_shared(st.q, proj, st.k, st.v, st.kvlen, *st.args(), True, st.segs, st.groups)
    want, _, tol, _ = st.attend()
    gate = torch.sigmoid(proj[:, :24 * 512].double().view(3, 24, 512)[..., 256:])
    want = want * gate
    assert ((out.view_as(want) - want).abs() <= (tol + 2.0 ** -20 * want.abs()) + 2.0 ** -8 * (want.abs() + tol)).all()


def test_rows_behind_the_last_segment_are_left_out(ops):
    st = shared_pages.Step(gen("behind"), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[9], [30, 31]])
    segs = tuple(t[:2] for t in st.segs[:3]) + (1,)
    ops.status_word.zero_()
    out = ops.attention_shared(st.q, None, st.k, st.v, st.kvlen, *st.args(), False, segs, st.groups)
    want, _, tol, _ = st.attend()
    assert ((out.view_as(want) - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol))[:2].all()
    mass = torch.zeros_like(st.mass)
    got = ops.attention_mass(st.q, st.k, mass, st.kvlen, *st.args(), segs, st.groups)
    assert abs(float(got.sum()) - 2 * 6) < 1e-3                          # two rows, a weight of one per head


def test_captured_steps_follow_their_tables(ops):
    """A captured call replayed with other lengths, pages and queries, and two captured calls that take turns."""
    g = gen("captured")
    kw = dict(groups=((300, [[400], [310], [555]]),), alone=[[70]])
    st = shared_pages.Step(g, DEV, 8, 2, 128, 64, poison=None, **kw)
    other = shared_pages.Step(gen("captured 2"), DEV, 8, 2, 128, 64, groups=((128, [[200], [450], [129]]),), alone=[[500]], poison=None)
    held = [t.clone() for t in (st.q, st.kvlen, st.table, *st.segs[:3], *st.groups)]
    side = torch.cuda.Stream()
    mass = st.mass.clone()

    def call():
        out, lse = attend(ops, st)
        return out, lse, ops.attention_mass(st.q, st.k, mass, st.kvlen, *st.args(), st.segs, st.groups, lse=lse, carry=0.0)
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = call()
        graphs.append((graph, res))
    for graph, (out, lse, sums) in graphs + graphs:
        graph.replay()
        torch.cuda.synchronize()
        check_attend(st, out, lse)
        want, tol, seen = st.masses(0.0)
        assert ((sums - want).abs() <= tol)[seen].all()
    st.q.copy_(other.q); st.kvlen.copy_(i32([333, 301, 400, 3]))
    other_view = shared_pages.Step.__new__(shared_pages.Step)
    other_view.__dict__.update(st.__dict__)
    other_view.streams, other_view.shared = [[333], [301], [400], [3]], [280]
    st.groups[2].copy_(i32([280]))
    for graph, (out, lse, sums) in graphs:
        graph.replay()
        torch.cuda.synchronize()
        check_attend(other_view, out, lse)
    for t, h in zip((st.q, st.kvlen, st.table, *st.segs[:3], *st.groups), held):
        t.copy_(h)


MANY = {
    "hundreds of streams": ([(200 + 7 * i, [[230 + 7 * i + j] for j in range(5)]) for i in range(30)], [[1 + i % 90] for i in range(170)]),
    "a thousand short ones": ([], [[1 + i % 3] for i in range(1000)]),
    "long rows among padding": ([(64, [[], [70], []]), (5, [[9]] * 9)], [[]] * 150 + [[2000, 1999], []]),
}


@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 64), (24, 1, 256), (8, 8, 128)])
@pytest.mark.parametrize("name", MANY)
def test_steps_of_many_streams(ops, name, nq, nkv, hd):
    """More streams than one pass of threads plans, and more blocks than a CTA keeps beside it."""
    groups, alone = MANY[name]
    st = shared_pages.Step(gen("many", name, nq), DEV, nq, nkv, hd, 64, groups, alone)
    out, lse = attend(ops, st)
    check_attend(st, out, lse)
    for known in (lse, None):
        check_mass(st, ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups, lse=known, carry=0.25, out=st.mass.clone()), 0.25)


@pytest.mark.parametrize("fill", [0x7fffffff, -1, 1 << 20])
def test_rows_of_refused_segments(ops, fill):
    """A segment that does not fit the step sets the status; its rows' places in the workspace were never written, whatever lies there, and the other rows are right."""
    for spoil in ("rows", "slot"):
        st = shared_pages.Step(gen("refused", spoil), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[9], [30, 31, 32], [77]])
        segs = st.segs
        if spoil == "rows":
            segs = (*segs[:3], 2)
        else:
            segs = (i32([*segs[0][:3].tolist(), -5, int(segs[0][4])]), *segs[1:])
        want, wl, tol, ltol = st.attend()
        ok = [0, 1, 2, 6]
        for lse_only in (False, True):
            n = ops.C.attention_shared_floats(st.rows, 5, segs[3], 1, 6, 2, 128, ops.sm_count, 0 if lse_only else 1)
            torch.full((n,), fill, dtype=torch.int32, device=DEV)      # what the allocator hands out next
            if lse_only:
                ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), segs, st.groups, out=st.mass.clone())
            else:
                out, lse = ops.attention_shared(st.q, None, st.k, st.v, st.kvlen, *st.args(), False, segs, st.groups, want_lse=True)
                assert ((out.view_as(want).double() - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30)[ok].all()
                assert ((lse - wl).abs() <= ltol)[ok].all()
            assert ops.status() != 0
            ops.status_word.zero_()


def test_padding_has_any_slot(ops):
    st = shared_pages.Step(gen("padding"), DEV, 6, 2, 128, 64, ((130, [[140], [], [200]]),), [[9], [], [77]])
    segs = (torch.where(st.segs[2] == 0, i32(-1), st.segs[0]).int(), *st.segs[1:])
    out, lse = ops.attention_shared(st.q, None, st.k, st.v, st.kvlen, *st.args(), False, segs, st.groups, want_lse=True)
    check_attend(st, out, lse)
    check_mass(st, ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), segs, st.groups, out=st.mass.clone()), 1.0)


def test_sums_of_a_pool_with_wide_tables(ops):
    """Tables with room for far more tokens than the pool has: the workspace follows the pool."""
    st = shared_pages.Step(gen("wide"), DEV, 4, 2, 64, 64, ((300, [list(range(290, 690)), [301]]),), [list(range(1, 500))], width=8000)
    assert ops.C.attention_mass_floats(st.rows, 3, 499, 1, 4, 2, 64, st.table.shape[1] * 64, st.k.shape[0] * 64, 0, ops.sm_count) < 1 << 23
    check_mass(st, ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups, out=st.mass.clone()), 1.0)


def test_large_pages_and_slots_that_come_twice(ops):
    """Two segments of one slot read the same pages, each with its own rows; pages of 1024 tokens."""
    st = shared_pages.Step(gen("twice"), DEV, 24, 4, 256, 1024, ((1500, [[1600, 1601], [1510]]),), [[2300, 2299], [40]])
    out, lse = attend(ops, st)
    check_attend(st, out, lse)
    slots, row0, nrows, most = st.segs                                  # the two rows of the third stream as a segment each
    twice = (i32([*slots[:3].tolist(), *slots[2:].tolist()]), i32([*row0[:3].tolist(), int(row0[2]) + 1, int(row0[3])]), i32([2, 1, 1, 1, 1]), most)
    out, lse = ops.attention_shared(st.q, None, st.k, st.v, st.kvlen, *st.args(), False, twice, st.groups, want_lse=True)
    check_attend(st, out, lse)


def test_pools_past_32_bits(ops):
    """A pool of more than 2^31 elements a cache: the bits of a small one with the same pages."""
    far, page, nkv, hd = 33200, 64, 4, 256
    small = shared_pages.Step(gen("far"), DEV, 24, nkv, hd, page, ((1200, [[1300], [1201, 1202]]),), [list(range(300, 700))], poison=None)
    n = small.k.shape[0]
    k, v = (torch.zeros(far, page, nkv, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    mass = torch.zeros(far, nkv, page, device=DEV)
    assert k.numel() > 1 << 31
    k[far - n:], v[far - n:], mass[far - n:] = small.k, small.v, small.mass
    table = torch.where(small.table >= 0, small.table + far - n, small.table)
    args = (table, *small.args()[1:])
    out, lse = attend(ops, small)
    far_out, far_lse = ops.attention_shared(small.q, None, k, v, small.kvlen, *args, False, small.segs, small.groups, want_lse=True)
    assert torch.equal(out, far_out) and torch.equal(lse, far_lse)
    for known in (lse, None):
        got = ops.attention_mass(small.q, small.k, small.mass, small.kvlen, *small.args(), small.segs, small.groups, lse=known, out=small.mass.clone())
        check_mass(small, got, 1.0)
        far_got = ops.attention_mass(small.q, k, mass, small.kvlen, *args, small.segs, small.groups, lse=known, out=mass.clone())
        assert torch.equal(got, far_got[far - n:])
    spare = sorted(set(range(n)) - set(small.table[small.table >= 0].tolist()))[:1]
    keep = page
    slot, length = small.segs[0][2:3], i32([699])
    kept = ops.kv_evict(small.k, small.v, None, small.mass, slot, length, small.table, i32([spare]), page, keep, 3, 20)
    far_kept = ops.kv_evict(k, v, None, mass, slot, length, table, i32([spare]) + far - n, page, keep, 3, 20)
    assert torch.equal(kept, far_kept)
    for a, b in ((small.k, k), (small.v, v), (small.mass, mass)):
        assert torch.equal(a, b[far - n:])


def test_two_streams_at_once(ops):
    sts = [shared_pages.Step(gen("stream", i), DEV, 24, 4, 256, 64, ((2000, [[2100 + i], [2500], [2001]]),), [[900]]) for i in range(2)]
    want = [attend(ops, st) for st in sts]
    sums = [ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups, lse=w[1], out=st.mass.clone()) for st, w in zip(sts, want)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sts]
    got = []
    for _ in range(5):
        for st, s, w in zip(sts, streams, want):
            with torch.cuda.stream(s):
                got.append((st, attend(ops, st), ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups, lse=w[1], out=st.mass.clone())))
    torch.cuda.synchronize()
    for st, (out, lse), m in got:
        i = sts.index(st)
        assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1]) and torch.equal(m, sums[i])


# ---- sums of weights --------------------------------------------------------------------------------------------------

def check_mass(st, got, carry, lse=None, start=None):
    want, tol, seen = st.masses(carry, lse, start)
    assert torch.equal(got[~seen], (st.mass if start is None else start)[~seen])
    bad = ~((got - want).abs() <= tol) & seen
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / tol)[seen].max()))


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("name", STEPS)
def test_sums(ops, name, nq, nkv, hd):
    groups, alone = STEPS[name]
    st = shared_pages.Step(gen("mass", name, nq, hd), DEV, nq, nkv, hd, {64: 192, 128: 64, 256: 64}[hd], groups, alone)
    _, lse = attend(ops, st)
    got = ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups, lse=lse, carry=0.5, out=st.mass.clone())
    check_mass(st, got, 0.5)
    empty = torch.where(st.spans().view(-1, 1, st.page), float("nan"), st.mass)       # not read
    got = ops.attention_mass(st.q, st.k, empty, st.kvlen, *st.args(), st.segs, st.groups, carry=0.0, out=st.mass.clone())
    check_mass(st, got, 0.0)
    mass = st.mass.clone()
    assert ops.attention_mass(st.q, st.k, mass, st.kvlen, *st.args(), st.segs, st.groups) is mass
    check_mass(st, mass, 1.0)


@pytest.mark.parametrize("nq,nkv,hd,lens", [(24, 4, 256, [(700, 300)]), (32, 8, 128, [(1111, 1111), (130, 33)]), (4, 2, 64, [(2000, 513), (64, 64)]),
                                            (6, 6, 128, [(600, 65)])])
def test_sums_of_prompts(ops, nq, nkv, hd, lens):
    """The last rows of prompts, with and without the logarithms in hand; the same bits every time."""
    st = shared_pages.Step(gen("prompt", nq, hd), DEV, nq, nkv, hd, 64, alone=[list(range(n - r + 1, n + 1)) for n, r in lens])
    got = [ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, carry=0.75, out=st.mass.clone()) for _ in range(2)]
    assert torch.equal(*got)
    check_mass(st, got[0], 0.75)
    _, lse = attend(ops, st)
    check_mass(st, ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, lse=lse, carry=0.75, out=st.mass.clone()), 0.75)


def test_sums_of_long_contexts(ops):
    st = shared_pages.Step(gen("mass long"), DEV, 24, 4, 256, 128, ((9000, [[9500], [9001], [12000]]),), [[30000]])
    check_mass(st, ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups, out=st.mass.clone()), 1.0)


# ---- eviction ---------------------------------------------------------------------------------------------------------

def pool(g, lens, keep, page, nkv, row, form, levels=None):
    need = [(n + page - 1) // page for n in lens]
    per = (keep + page - 1) // page
    total = sum(need) + len(lens) * per + 2
    order = torch.randperm(total, generator=g, device=DEV).int()
    table, at = torch.full((len(lens) + 1, max(need + [1]) + 1), -1, dtype=torch.int32, device=DEV), 0
    for s, k in enumerate(need):
        table[s + 1, :k] = order[at:at + k]
        at += k
    dst = order[at:at + len(lens) * per].view(len(lens), per).contiguous()
    scale = None
    if form == "bf16":
        k, v = (torch.randn(total, page, nkv, row, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    else:
        k, v = (torch.randint(0, 256, (total, page, nkv, row), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2))
        scale = torch.randn(total, page, nkv, {"fp8": 2, "int4": 16, "int6": 4}[form], generator=g, device=DEV)
    if levels:
        mass = torch.randint(0, levels, (total, nkv, page), generator=g, device=DEV).float()
    else:
        mass = torch.randn(total, nkv, page, generator=g, device=DEV).exp()
    return table, dst, k, v, scale, mass


def check_evict(ops, lens, keep, first, recent, page, nkv, table, dst, k, v, scale, mass):
    old = [x.clone() if x is not None else None for x in (k, v, scale, mass)]
    slots = i32([s + 1 for s in range(len(lens))])
    kept = ops.kv_evict(k, v, scale, mass, slots, i32(lens), table, dst, page, keep, first, recent)
    want = [x.clone() if x is not None else None for x in old]
    for s, n in enumerate(lens):
        pages = table[s + 1].cpu()
        for h in range(nkv):
            w = old[3][pages[:(n + page - 1) // page].long().to(DEV), h].reshape(-1)[:n].tolist()
            ids = shared_pages.evicted(w, n, keep, first, recent)
            assert kept[s, h].tolist() == ids + [-1] * (keep - len(ids))
            j = torch.tensor(ids, dtype=torch.long, device=DEV)
            i = torch.arange(len(ids), device=DEV)
            a, b, c, d = table[s + 1].long()[j // page], j % page, dst[s].long()[i // page], i % page
            for x, was in zip(want[:3], old[:3]):
                if x is not None:
                    x[c, d, h] = was[a, b, h]
            want[3][c, h, d] = old[3][a, h, b]
    for x, w in zip((k, v, scale, mass), want):                          # nothing else moved
        if x is not None:
            assert torch.equal(x.view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("form,row", [("bf16", 256), ("bf16", 64), ("fp8", 256), ("int4", 32), ("int6", 48)])
@pytest.mark.parametrize("lens,keep,first,recent,page", [([500, 64, 0, 700, 129], 128, 4, 32, 64), ([1, 2], 1, 0, 0, 64), ([300], 70, 0, 70, 16),
                                                         ([257, 1000], 200, 7, 0, 1), ([90, 91], 91, 1, 5, 192)])
def test_evict(ops, form, row, lens, keep, first, recent, page):
    g = gen("evict", form, keep)
    check_evict(ops, lens, keep, first, recent, page, 3, *pool(g, lens, keep, page, 3, row, form))


@pytest.mark.parametrize("levels", [1, 2, 5])
def test_evict_of_equal_weights(ops, levels):
    lens = [3000, 1025, 5000]
    check_evict(ops, lens, 1024, 4, 100, 64, 2, *pool(gen("equal", levels), lens, 1024, 64, 2, 64, "bf16", levels))


def test_evict_of_odd_weights(ops):
    """No numbers count as the largest, zeros of both signs are equal, infinities, numbers below the normal ones."""
    lens = [2000, 777]
    p = pool(gen("odd"), lens, 300, 64, 2, 64, "bf16")
    m = p[-1]
    r = torch.rand(m.shape, generator=gen("odd places"), device=DEV)
    for lo, val in ((0.0, float("nan")), (0.02, float("inf")), (0.04, -float("inf")), (0.06, 0.0), (0.4, -0.0), (0.8, 1e-41), (0.85, -1e-41), (0.9, 3e38)):
        m[r >= lo] = val
    check_evict(ops, lens, 300, 3, 50, 64, 2, *p)


def test_evict_of_a_long_context(ops):
    lens = [100000, 33333]
    check_evict(ops, lens, 8192, 16, 1000, 64, 2, *pool(gen("evict long"), lens, 8192, 64, 2, 256, "fp8"))


# ---- one after the other ----------------------------------------------------------------------------------------------

def test_a_server_shrinks_its_contexts(ops):
    """Attention over a shared prefix, sums of its weights, eviction by them, attention over what stayed."""
    nq, nkv, hd, page, keep = 8, 2, 128, 64, 256
    st = shared_pages.Step(gen("chain"), DEV, nq, nkv, hd, page, ((640, [[900], [700], [1000]]),), [[333]], spare=4 * 4 + 2, poison=None, q_scale=2.0)
    mass = torch.zeros_like(st.mass)
    for _ in range(2):
        out, lse = attend(ops, st)
        ops.attention_mass(st.q, st.k, mass, st.kvlen, *st.args(), st.segs, st.groups, lse=lse)
    want, tol, seen = st.masses(0.0)
    assert ((mass - 2 * want).abs() <= 2 * tol + 2.0 ** -22 * want)[seen].all()
    used = torch.zeros(st.k.shape[0], dtype=torch.bool, device=DEV)
    used[st.table[st.table >= 0].long()] = True
    dst = torch.nonzero(~used).flatten()[:16].int().view(4, 4).contiguous()
    lens = [900, 700, 1000, 333]
    held = mass.clone()
    kept = ops.kv_evict(st.k, st.v, None, mass, i32(st.slots), i32(lens), st.table, dst, page, keep, 4, 64)
    for s, n in enumerate(lens):
        for h in range(nkv):
            w = held[st.table[s, torch.arange(n, device=DEV) // page].long(), h, torch.arange(n, device=DEV) % page].tolist()
            assert kept[s, h].tolist() == shared_pages.evicted(w, n, keep, 4, 64)
    out = ops.attention_shared(st.q, None, st.k, st.v, i32([keep] * 4), dst, page, nq, nkv, hd, False, st.segs)
    for s in range(4):
        for h in range(nkv):
            at = st.table[s].long()[kept[s, h].long() // page] * page + kept[s, h].long() % page
            k, v = st.k.view(-1, nkv, hd)[at, h].double(), st.v.view(-1, nkv, hd)[at, h].double()
            q = st.q[s].view(nkv, -1, hd)[h].double()
            p = torch.softmax(q @ k.t() / hd ** 0.5, -1)
            want = p @ v
            tol = p @ v.abs() * (2 * (2.0 ** -20 * (q.abs() @ k.abs().t() / hd ** 0.5).max() + 2.0 ** -20) + 2.0 ** -8)
            got = out.view(4, nkv, -1, hd)[s, h].double()
            assert ((got - want).abs() <= tol + 2.0 ** -8 * (want.abs() + tol)).all()


# ---- refusals ---------------------------------------------------------------------------------------------------------

def test_refusals(ops):
    st = shared_pages.Step(gen("refuse"), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[9]])
    base = dict(q=st.q, proj=None, k_cache=st.k, v_cache=st.v, row_kvlen=st.kvlen, block_table=st.table, kv_block=64, nq=6, nkv=2, hd=128, gated=False,
                segs=st.segs, groups=st.groups)
    odd = torch.zeros(4, 32, 2, 128, dtype=torch.bfloat16, device=DEV)
    for change in (dict(q=st.q.half()), dict(k_cache=st.k.float()), dict(v_cache=st.v[:1]), dict(k_cache=odd, v_cache=odd, kv_block=32), dict(nq=5, q=st.q[:, :5]),
                   dict(hd=96), dict(row_kvlen=st.kvlen.long()), dict(row_kvlen=st.kvlen[:2]), dict(block_table=st.table.t()), dict(block_table=st.table.cpu()),
                   dict(segs=(st.segs[0][:2], *st.segs[1:])), dict(gated=True, proj=torch.zeros(3, 100, dtype=torch.bfloat16, device=DEV)),
                   dict(groups=(st.groups[0], st.groups[1], st.groups[2].float())), dict(k_cache=st.k.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(RuntimeError):
            ops.attention_shared(**{**base, **change})
    with pytest.raises(RuntimeError):
        ops.attention_shared(**{**base, "gated": True})                # no proj
    many = 4097
    with pytest.raises(RuntimeError):
        ops.attention_shared(**{**base, "segs": (*(torch.zeros(many, dtype=torch.int32, device=DEV) for _ in range(3)), 1), "groups": None})
    with pytest.raises(RuntimeError):
        ops.attention_mass(torch.zeros(3, 130, 128, dtype=torch.bfloat16, device=DEV), st.k, st.mass, st.kvlen, st.table, 64, 130, 2, 128, st.segs, st.groups)   # share 65
    mbase = dict(q=st.q, k_cache=st.k, mass=st.mass, row_kvlen=st.kvlen, block_table=st.table, kv_block=64, nq=6, nkv=2, hd=128, segs=st.segs, groups=st.groups)
    for change in (dict(mass=st.mass.half()), dict(mass=st.mass.transpose(1, 2).contiguous()), dict(out=st.mass[:1]), dict(lse=torch.zeros(2, 6, device=DEV)),
                   dict(lse=torch.zeros(3, 6, device=DEV, dtype=torch.bfloat16)), dict(k_cache=st.k.float())):
        with pytest.raises(RuntimeError):
            ops.attention_mass(**{**mbase, **change})
    p = pool(gen("refuse evict"), [100], 32, 64, 2, 64, "bf16")
    table, dst, k, v, scale, mass = p
    ebase = dict(k_cache=k, v_cache=v, kv_scale=None, mass=mass, seg_slot=i32([1]), seg_len=i32([100]), block_table=table, dst_table=dst, kv_block=64, keep=32)
    for change in (dict(keep=0), dict(keep=65), dict(first=20, recent=13), dict(first=-1), dict(recent=-1), dict(kv_block=32), dict(v_cache=v.half()),
                   dict(mass=mass.double()), dict(kv_scale=torch.zeros(1, device=DEV)), dict(seg_len=i32([100, 1])), dict(dst_table=dst[:0]),
                   dict(k_cache=k[..., :4].contiguous(), v_cache=v[..., :4].contiguous())):
        with pytest.raises(RuntimeError):
            ops.kv_evict(**{**ebase, **change})


def test_tables_that_are_wrong_are_reported(ops):
    """A page that is none and a context beyond the table set the status; nothing outside the pool is touched."""
    for spoil in ("page", "far page", "length", "slot", "group"):
        st = shared_pages.Step(gen("wrong", spoil), DEV, 6, 2, 128, 64, ((130, [[140], [200]]),), [[9]])
        assert ops.status() == 0
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
        attend(ops, st)
        torch.cuda.synchronize()
        assert ops.status() != 0, spoil
        ops.status_word.zero_()
        ops.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups)
        assert ops.status() != 0, spoil
        ops.status_word.zero_()
    table, dst, k, v, scale, mass = pool(gen("wrong evict"), [200], 64, 64, 2, 64, "bf16")
    for spoil in ("page", "dst", "length", "slot"):
        t, d, n, slot = table.clone(), dst.clone(), i32([200]), i32([1])
        if spoil == "page":
            t[1, 2] = 1 << 20
        elif spoil == "dst":
            d[0, 0] = -1
        elif spoil == "length":
            n = i32([1 << 20])
        else:
            slot = i32([-1])
        ops.kv_evict(k, v, scale, mass, slot, n, t, d, 64, 64)
        assert ops.status() != 0, spoil
        ops.status_word.zero_()
