"""Ops over a page pool that streams share, on the CPU: the plain statement against 64 bits, and what it refuses."""
import pytest
import shared_pages
import torch

from ferrite_b200.ops.torch_ops import TorchOps

OPS = TorchOps()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def step(seed, **kw):
    base = dict(nq=6, nkv=2, hd=16, page=8, groups=[(21, [[25, 26], [22], [21, 0]]), (8, [[9], [3]])], alone=[[13], [1, 2, 3]], dtype=torch.float32)
    return shared_pages.Step(gen(seed), "cpu", **{**base, **kw})


@pytest.mark.parametrize("groups,alone", [(((21, [[25, 26], [22], [21, 0]]), (8, [[9], [3]])), [[13], [1, 2, 3]]), ((), [[40], [7, 5]]), (((0, [[5], [6]]),), []),
                                          (((64, [[64]]),), [])])
def test_attention_and_sums(groups, alone):
    st = step(1, groups=groups, alone=alone)
    out, lse = OPS.attention_shared(st.q, None, st.k, st.v, st.kvlen, *st.args(), False, st.segs, st.groups, want_lse=True)
    want, wl, tol, ltol = st.attend()
    assert ((out.view_as(want) - want).abs() <= tol + 1e-6).all()
    assert torch.equal(torch.isinf(lse), torch.isinf(wl)) and ((lse - wl).nan_to_num(0, 0, 0).abs() <= ltol + 1e-6).all()
    for given in (None, lse):
        for carry in (0.0, 0.5, 1.0):
            mass = st.mass.clone()
            if carry == 0:
                mass[:] = float("nan")                                # not read
            got = OPS.attention_mass(st.q, st.k, mass, st.kvlen, *st.args(), st.segs, st.groups, lse=given, carry=carry, out=st.mass.clone())
            want, tol, seen = st.masses(carry)
            assert ((got - want).abs() <= tol + 1e-6).all()
            assert torch.equal(got[~seen], st.mass[~seen])
    mass = st.mass.clone()
    assert OPS.attention_mass(st.q, st.k, mass, st.kvlen, *st.args(), st.segs, st.groups) is mass


def test_gate():
    st = step(2)
    proj = torch.randn(st.rows, st.nq * 2 * st.hd + 5, generator=gen(3))
    plain = OPS.attention_shared(st.q, proj, st.k, st.v, st.kvlen, *st.args(), False, st.segs, st.groups)
    gated = OPS.attention_shared(st.q, proj, st.k, st.v, st.kvlen, *st.args(), True, st.segs, st.groups)
    gate = torch.sigmoid(proj[:, :st.nq * 2 * st.hd].view(st.rows, st.nq, 2 * st.hd)[..., st.hd:]).reshape(st.rows, -1)
    assert torch.allclose(gated, plain * gate, atol=1e-6)


def test_sums_of_a_step_are_the_rows_that_saw_something():
    """Weights of a row add up to one per head, wherever its keys lie."""
    st = step(4)
    got = OPS.attention_mass(st.q, st.k, torch.zeros_like(st.mass), st.kvlen, *st.args(), st.segs, st.groups)
    rows = int((st.kvlen > 0).sum())
    assert torch.allclose(got.sum((0, 2)), torch.full((st.nkv,), float(rows * st.nq // st.nkv)), rtol=1e-5)


@pytest.mark.parametrize("lens,keep,first,recent,page", [([40, 7, 0, 12], 12, 2, 3, 4), ([9], 9, 0, 0, 8), ([33, 34], 5, 0, 5, 16), ([20], 1, 0, 0, 1),
                                                         ([50], 7, 3, 0, 8)])
def test_evict(lens, keep, first, recent, page):
    g = gen(5)
    need = [(n + page - 1) // page for n in lens]
    dst_pages = (keep + page - 1) // page
    total = sum(need) + len(lens) * dst_pages + 1
    order = torch.randperm(total, generator=g).int()
    table, at = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32), 0
    for s, k in enumerate(need):
        table[s, :k] = order[at:at + k]
        at += k
    dst = order[at:at + len(lens) * dst_pages].view(len(lens), -1)
    k, v = torch.randn(total, page, 3, 8, generator=g), torch.randn(total, page, 3, 8, generator=g)
    scale = torch.randn(total, page, 3, 2, generator=g)
    mass = torch.randint(0, 4, (total, 3, page), generator=g).float()                 # many equal ones
    mass[torch.rand(mass.shape, generator=g) < 0.05] = float("nan")
    old = [x.clone() for x in (k, v, scale, mass)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    kept = OPS.kv_evict(k, v, scale, mass, i32(list(range(len(lens)))), i32(lens), table, dst, page, keep, first, recent)
    for s, n in enumerate(lens):
        for h in range(3):
            w = [float(old[3][table[s, j // page], h, j % page]) for j in range(n)]
            ids = shared_pages.evicted(w, n, keep, first, recent)
            assert kept[s, h].tolist() == ids + [-1] * (keep - len(ids))
            for i, j in enumerate(ids):
                a, b = (int(table[s, j // page]), j % page), (int(dst[s, i // page]), i % page)
                for new, was in zip((k, v, scale), old):
                    assert torch.equal(new[b[0], b[1], h], was[a[0], a[1], h])
                assert torch.equal(mass[b[0], h, b[1]].nan_to_num(-1), old[3][a[0], h, a[1]].nan_to_num(-1))


def test_evict_refuses():
    z = torch.zeros(4, 8, 2, 16)
    one = torch.ones(1, dtype=torch.int32)
    for keep, first, recent in ((0, 0, 0), (9, 0, 0), (4, 3, 2), (4, -1, 0), (4, 0, -1)):
        with pytest.raises(RuntimeError):
            OPS.kv_evict(z, z, None, torch.zeros(4, 2, 8), one, one, one[None], one[None], 8, keep, first, recent)


def test_sums_refuse_keys_that_two_segments_hold():
    """Streams that were forked twice, a slot that comes twice, a page that comes twice in a table: a key's sum is written once."""
    for spoil in ("forked twice", "slot", "page"):
        st = step(6, groups=[(16, [[17], [41], [45]])], alone=[[33]])
        if spoil == "forked twice":
            st.table[2, 2:4] = st.table[1, 2:4]
        elif spoil == "slot":
            st.segs[0][3] = 2
        else:
            st.table[3, 3] = st.table[3, 1]
        with pytest.raises(RuntimeError):
            OPS.attention_mass(st.q, st.k, st.mass, st.kvlen, *st.args(), st.segs, st.groups)
    st = step(6, groups=[(16, [[17], [41], [45]])], alone=[[33]])
    st.table[2, 2:4] = st.table[1, 2:4]                                   # one by one
    whole = torch.zeros_like(st.mass)
    for s in range(4):
        segs = tuple(t[s:s + 1] for t in st.segs[:3]) + (1,)
        OPS.attention_mass(st.q, st.k, whole, st.kvlen, *st.args(), segs)
    assert torch.allclose(whole.sum((0, 2)), torch.full((2,), 4.0 * 3), rtol=1e-5)
