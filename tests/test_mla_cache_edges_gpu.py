"""Latents in 4 and 8 bits where steps, pages and values go to their limits."""
import latent_rows as lr
import pytest
import torch
from test_mla_cache_gpu import DEV, R, bf, check_attention, clean, gen, i32, inv_freq, ops, random_cache, segments, tables  # noqa: F401

from ferrite_b200.ops import mla_cache

pytestmark = pytest.mark.gpu


def key_parts(cache, table, slot, page, L, bits, first):
    """The key parts of a stream's rows: `first` [n] ahead, zeros behind."""
    p = torch.arange(len(first), device=DEV)
    flat = table[slot, p // page].long() * page + p % page
    rope = torch.zeros(len(first), R, dtype=torch.bfloat16, device=DEV)
    rope[:, 0] = first
    at = L * bits // 8
    cache.view(-1, cache.shape[-1])[flat, at:at + 2 * R] = rope.view(torch.uint8).view(len(first), 2 * R)
    return flat


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nq", [16, 128])
@pytest.mark.parametrize("far", [-60.0, 60.0])
def test_a_piece_that_is_no_number_is_not_lost(ops, bits, nq, far):
    """Keys that CTAs of their own attend, one of them (`far` below the others) or all of the first CTA's (the others `far` above) no number: every score
    is in the softmax, so the row is no number, however little such keys would weigh."""
    g = gen("piece", bits, nq, far)
    L, n, page = 512, 512, 64
    table, pages = tables([n], page, g)
    cache = random_cache(bits, L, pages, page, g)
    first = torch.zeros(n, device=DEV)
    first[:128] = far if far < 0 else 0
    first[128:] = 0 if far < 0 else far
    flat = key_parts(cache, table, 0, page, L, bits, first)
    q = bf(g, 1, nq, L + R, sc=0.2)
    q[..., L] = 100                                                    # 433 in log2 between the two
    check_attention(ops, bits, L, nq, page, [0], [n], table, cache, q, 0.05, segments(1, 1))
    bad = flat[5:6] if far < 0 else flat[:128]
    cache.view(-1, cache.shape[-1])[bad, L * bits // 8 + 2 * R + 3] = 255
    got = ops.mla_attention(q, cache, i32([0]), i32([n]), table, page, nq, L, R, 0.05, segs=segments(1, 1), kv_bits=bits)
    assert got.isnan().all()


@pytest.mark.parametrize("bits", [4, 8])
def test_a_key_that_is_no_number_is_not_lost_when_scores_rise(ops, bits):
    """The same inside a CTA's piece: a key that is none in its first tile, scores 433 higher (log2) in its second, and as much higher again elsewhere."""
    g = gen("rise", bits)
    L, page, nq = 512, 64, 16
    n = 2 * 128 * ops.sm_count                                         # two tiles a CTA
    table, pages = tables([n], page, g)
    cache = random_cache(bits, L, pages, page, g)
    first = torch.full((n,), 60.0, device=DEV)
    first[:128], first[128:256] = -60, 0
    flat = key_parts(cache, table, 0, page, L, bits, first)
    q = bf(g, 1, nq, L + R, sc=0.2)
    q[..., L] = 100
    call = lambda: ops.mla_attention(q, cache, i32([0]), i32([n]), table, page, nq, L, R, 0.05, segs=segments(1, 1), kv_bits=bits)
    assert call().isfinite().all()
    cache.view(-1, cache.shape[-1])[flat[7], L * bits // 8 + 2 * R] = 255
    assert call().isnan().all()


@pytest.mark.parametrize("bits", [4, 8])
def test_segments_of_more_rows_than_said_leave_the_output_alone(ops, bits):
    """A workspace that an earlier call has used, and a segment of five rows where one was said: the status says so and nothing is written."""
    g = gen("capacity", bits)
    L, nq, page, n, T = 512, 16, 64, 1000, 5
    table, pages = tables([n], page, g)
    cache = random_cache(bits, L, pages, page, g)
    q, out = bf(g, T, nq, L + R), torch.full((T, nq, L), 7.0, dtype=torch.bfloat16, device=DEV)
    ws = torch.zeros(ops.C.mla_attn_q_floats(1, nq, L, ops.sm_count), device=DEV)
    call = lambda rows: ops.C.mla_attn_q(out, ws, q, cache, i32([0]), i32([0]), i32([rows]), 1, i32([n] * T), table, page, L, R, bits, 0.05, ops.sm_count,
                                         ops.status_word)
    call(1)
    assert ops.status() == 0 and not (out[0] == 7).any() and (out[1:] == 7).all()
    out.fill_(7)
    call(T)
    assert ops.status() == 5
    ops.status_word.zero_()
    assert (out == 7).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_prep_takes_eps_in_64_bits(ops, bits):
    """A row whose mean square is about eps: mean square + eps is 2^-18 (1 + 2^-30), so a value that would lie on the border of two codes (3.5 of 4 bits;
    15.5 of e4m3) lies below it, by less than eps has in 32 bits."""
    L, nq, dn, page = 64, 2, 32, 64
    u = 2.0 ** -9
    kva = torch.zeros(1, L + R, dtype=torch.bfloat16, device=DEV)
    kva[0, :3] = torch.tensor([7.0, 3.5, 31 / 128]) * u
    eps = u * u * (1 + 2.0 ** -30) - float(kva[0, :L].double().square().sum()) / L
    assert float(torch.tensor(eps)) != eps
    w, q = torch.zeros(L, dtype=torch.bfloat16, device=DEV), torch.zeros(1, nq * (dn + R), dtype=torch.bfloat16, device=DEV)
    cache = torch.zeros(1, page, lr.row_bytes(L, bits), dtype=torch.uint8, device=DEV)
    ops.mla_prep(q, kva, w, None, inv_freq(), i32([0]), i32([0]), i32([[0]]), cache, page, nq, dn, L, R, eps, absorb=False, kv_bits=bits)
    want = mla_cache.quantised(lr.normed(kva, w, L, eps), bits).cpu()
    assert want[0, 1 if bits == 4 else 2] == (3.0 if bits == 4 else 15 / 64)
    assert torch.equal(lr.unpack(cache[0, :1], L, bits)[:, :L], want)
