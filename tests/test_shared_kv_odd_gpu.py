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
