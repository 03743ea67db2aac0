"""Latents in 4 and 8 bits where steps, pages and values go to their limits."""
import dataclasses

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


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_of_a_prompt_walk_tiles_of_their_own_contexts(ops, bits):
    """A causal segment of 140 rows, 64 heads: a unit is a row, and walks as many tiles as the last row of its 64 sees. The CTAs share the tiles, and a place
    more for each unit, evenly. What the kernel leaves for the join says in which CTA each unit starts and ends."""
    g = gen("units", bits)
    L, nq, page, rows, ctas = 64, 64, 64, 140, ops.sm_count
    assert rows <= ctas
    table, pages = tables([128 * rows], page, g)
    cache = random_cache(bits, L, pages, page, g)
    kvlen = [128 * (r + 1) for r in range(rows)]
    q, out = bf(g, rows, nq, L + R), torch.empty(rows, nq, L, dtype=torch.bfloat16, device=DEV)
    segs = (i32([0]), i32([0]), i32([rows]), rows)
    ws = torch.zeros(ops.C.mla_attn_q_floats(rows, nq, L, ctas), device=DEV)
    ops.C.mla_attn_q(out, ws, q, cache, *segs, i32(kvlen), table, page, L, R, bits, 0.1, ctas, ops.status_word)
    jobs = ws[:4 * rows].view(torch.int32).view(rows, 4).cpu()
    own = [min(rows, r // 64 * 64 + 64) for r in range(rows)]              # tiles of a row's unit
    start = [sum(n + 1 for n in own[:r]) for r in range(rows)]
    share = -(-(start[-1] + own[-1] + 1) // ctas)
    assert jobs[:, 0].tolist() == [r * nq for r in range(rows)]
    assert (jobs[:, 2] // 2).tolist() == [s // share for s in start]
    assert jobs[:, 3].tolist() == [(s + n - 1) // share for s, n in zip(start, own)]
    assert torch.equal(out, check_attention(ops, bits, L, nq, page, [0] * rows, kvlen, table, cache, q, 0.1, segs))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nq", [128, 16, 3, 1])
@pytest.mark.parametrize("width", [0, 300])
def test_attention_of_prompts_on_small_pages(ops, bits, nq, width):
    """Causal segments of hundreds of rows beside short ones and single rows, on pages of 24 tokens."""
    g = gen("prompts", bits, nq, width)
    lens, nrows, L = [700, 90, 333, 0, 20, 512], [400, 1, 333, 0, 5, 40], 64
    table, pages = tables(lens, 24, g, width=width)
    cache = random_cache(bits, L, pages, 24, g)
    slot = [s for s, r in enumerate(nrows) for _ in range(r)]
    kvlen = [lens[s] - r + 1 + i for s, r in enumerate(nrows) for i in range(r)]
    row0 = [sum(nrows[:s]) for s in range(len(nrows))]
    check_attention(ops, bits, L, nq, 24, slot, kvlen, table, cache, bf(g, len(slot), nq, L + R), (L + R) ** -0.5,
                    (i32(list(range(len(nrows)))), i32(row0), i32(nrows), max(nrows)))


@pytest.mark.parametrize("latent", [64, 512])
@pytest.mark.parametrize("kv", ["int4", "fp8"])
def test_engine_prompts_on_small_pages(ext, kv, latent):
    """Pages of 16 tokens: prompts take the absorbed form, causal rows over codes; against the CPU engine over the same format, as near as the expanded
    form on pages of 64 has to be."""
    from ferrite_b200.config import EngineConfig, tiny_mla
    from ferrite_b200.engine.engine import Engine
    from ferrite_b200.engine.executor import Segment
    from ferrite_b200.models.weights import init_weights
    cfg = dataclasses.replace(tiny_mla(), kv_lora=latent)
    w = init_weights(cfg, seed=0)
    p = torch.randint(0, cfg.vocab, (200,), generator=torch.Generator().manual_seed(4)).tolist()
    want = Engine(cfg, w, EngineConfig(n_slots=1, max_ctx=256, kv_dtype=kv), device="cpu").forward([Segment(0, 0, p, "all")])[0]
    eng = Engine(cfg, w, EngineConfig(n_slots=1, max_ctx=256, kv_dtype=kv, kv_block=16), device=DEV)
    got = torch.cat([eng.forward([Segment(0, 0, p[:150], "all")])[0].clone(), eng.forward([Segment(0, 150, p[150:], "all")])[0].clone()]).float().cpu()
    eng.check()
    kl = torch.nn.functional.kl_div(torch.log_softmax(got, -1), torch.log_softmax(want, -1), log_target=True, reduction="batchmean").item()
    assert kl < (8e-2 if kv == "int4" else 3e-2), kl


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("nq", [128, 16, 3])
@pytest.mark.parametrize("width", [0, 300])
@pytest.mark.parametrize("rows", [17, 150])
def test_rows_of_a_segment_in_any_order(ops, bits, nq, width, rows):
    """Contexts that fall along a segment, or come in no order, some of them empty."""
    g = gen("order", bits, nq, width, rows)
    lens, L = [700, 300, 130], 512 if rows == 17 else 64
    table, pages = tables(lens, 64, g, width=width)
    cache = random_cache(bits, L, pages, 64, g)
    slot = [s for s in range(3) for _ in range(rows)]
    kvlen = [700 - 600 * r // rows for r in range(rows)]
    kvlen += torch.randint(0, 301, (rows,), generator=torch.Generator().manual_seed(nq)).tolist()
    kvlen += [130 if r % 3 == 1 else 0 if r % 3 == 0 else 129 for r in range(rows)]
    check_attention(ops, bits, L, nq, 64, slot, kvlen, table, cache, bf(g, 3 * rows, nq, L + R), 0.05, segments(rows, 3))


@pytest.mark.parametrize("rows", [3, 90])
@pytest.mark.parametrize("at", [0, 1, -1])
def test_any_row_that_sees_past_the_table_sets_the_status(ops, rows, at):
    g = gen("past", rows, at)
    table, pages = tables([128], 64, g)
    cache = random_cache(4, 64, pages, 64, g)
    kvlen = [100] * rows
    kvlen[at] = 200
    ops.mla_attention(bf(g, rows, 4, 64 + R), cache, i32([0] * rows), i32(kvlen), table, 64, 4, 64, R, 0.05, segs=segments(rows, 1), kv_bits=4)
    assert ops.status() == 3
    ops.status_word.zero_()


def bounds(bits, L, page, slot, kvlen, table, cache, q, scale):
    """How far `check_attention` lets every output be from 64 bits."""
    vals = lr.unpack(cache.view(-1, cache.shape[-1]), L, bits).to(DEV)
    out = []
    for r, (s, n) in enumerate(zip(slot, kvlen)):
        p = torch.arange(n, device=DEV)
        keys, qr = vals[table[s, p // page].long() * page + p % page], q[r].double()
        w = torch.softmax(qr @ keys.t() * scale, -1)
        ds = (qr.abs() @ keys.abs().t() * scale).amax(-1, keepdim=True) * (L + R) / 16 * 2 ** -23
        out.append(2 ** -8 * (w @ keys[:, :L]).abs() + (w @ keys[:, :L].abs()) * (2 ** -11 + 2 * ds) + 1e-30)
    return torch.stack(out)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("L,nq", [(512, 128), (512, 16), (64, 4)])
@pytest.mark.parametrize("first", [30, 2040])
def test_how_far_a_row_moves_from_step_to_step(ops, bits, L, nq, first):
    """A row decoded alone, verified among seventeen and beside other streams: its keys are cut at other places, so it may round differently. Each is within
    `check_attention`'s distance of 64 bits, so two of them are within twice that of each other; the same step again gives the same bits."""
    g = gen("moves", bits, L, nq, first)
    rows, lens, page = 17, [first + 17, 60, 5000], 64
    table, pages = tables(lens, page, g)
    cache = random_cache(bits, L, pages, page, g)
    q, scale = bf(g, rows + 2, nq, L + R), (L + R) ** -0.5

    def step(parts):                                         # (stream, first row, rows) of each segment
        at = [r for _, r, n in parts for r in range(r, r + n)]
        own = [first + 1 + r if s == 0 else lens[s] for s, a, n in parts for r in range(a, a + n)]
        slot, row0 = [s for s, _, n in parts for _ in range(n)], [sum(n for _, _, n in parts[:i]) for i in range(len(parts))]
        segs = (i32([s for s, _, _ in parts]), i32(row0), i32([n for _, _, n in parts]), max(n for _, _, n in parts))
        got = check_attention(ops, bits, L, nq, page, slot, own, table, cache, q[at], scale, segs)
        again = ops.mla_attention(q[at], cache, i32(slot), i32(own), table, page, nq, L, R, scale, segs=segs, kv_bits=bits)
        assert torch.equal(got, again)
        return got.double()

    tol = 2 * bounds(bits, L, page, [0] * rows + [1, 2], list(range(first + 1, first + rows + 1)) + lens[1:], table, cache, q, scale)
    whole = step([(0, 0, rows)])
    beside = step([(1, rows, 1), (0, 0, rows), (2, rows + 1, 1)])
    assert ((beside[1:1 + rows] - whole).abs() <= tol[:rows]).all()
    for r in (0, 8, 16):
        assert ((step([(0, r, 1)])[0] - whole[r]).abs() <= tol[r]).all()
    assert ((step([(1, rows, 1)])[0] - beside[0]).abs() <= tol[rows]).all() and ((step([(2, rows + 1, 1)])[0] - beside[-1]).abs() <= tol[rows + 1]).all()


@pytest.mark.parametrize("latent", [64, 512])
@pytest.mark.parametrize("kv", ["int4", "fp8"])
def test_engine_row_alone_beside_others_and_verified(ext, kv, latent):
    """A token behind the same context, decoded alone, beside other streams and as the first of verified rows, and the rows behind it against decoding
    them one by one. Only the step's own rows can differ (bf16 roundings of its products, its cuts of the keys, its own latents' codes next to a border):
    less than what holding ALL latents of the context in codes instead of 16 bits changes."""
    from ferrite_b200.config import EngineConfig, tiny_mla
    from ferrite_b200.engine.engine import Engine
    from ferrite_b200.engine.executor import Segment
    from ferrite_b200.models.weights import init_weights
    cfg = dataclasses.replace(tiny_mla(moe=False), kv_lora=latent)
    w = init_weights(cfg, seed=0)
    g = torch.Generator().manual_seed(3)
    p, other, new = (torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (300, 60, 5))

    def run(kv):
        eng = Engine(cfg, w, EngineConfig(n_slots=5, max_ctx=512, kv_dtype=kv), device=DEV)
        eng.forward([Segment(0, 0, p, "none")])
        eng.forward([Segment(4, 0, other, "none")])
        for s in (1, 2, 3):
            eng.ex.copy_slot(0, s, len(p))
        alone = torch.cat([eng.forward([Segment(1, 300 + i, [t], "last")])[0].clone() for i, t in enumerate(new)])
        beside = eng.forward([Segment(4, 60, [7], "last"), Segment(2, 300, [new[0]], "last"), Segment(0, 300, [9], "last")])[0].clone()
        verified = eng.forward([Segment(3, 300, new, "all")], commit=False)[0].clone()
        eng.check()
        return alone.double(), beside[1].double(), verified.double()

    alone, beside, verified = run(kv)
    format_moves = (alone - run("bf16")[0]).norm(dim=1)
    assert (format_moves > 0).all()
    assert (beside - alone[0]).norm() <= format_moves[0]
    assert ((verified - alone).norm(dim=1) <= format_moves).all()


@pytest.mark.parametrize("ctas", [1, 7, 61, 148])
@pytest.mark.parametrize("nq,n", [(16, 9), (3, 45), (40, 45)])
def test_prompts_and_single_rows_cut_anywhere(ops, nq, n, ctas, monkeypatch):
    """Prompts of up to 200 rows among single and verified rows, more segments than a warp has lanes, shared out over few CTAs and many."""
    g = gen("cut", nq, n)
    L, page = 64, 24
    nrows = [0 if i % 7 == 3 else 65 + 27 * (i % 6) if i % 4 == 1 else 1 + i % 5 for i in range(n)]
    lens = [r + (i * 53) % 150 for i, r in enumerate(nrows)]
    table, pages = tables(lens, page, g, width=11 * (nq == 16))
    cache = random_cache(4, L, pages, page, g)
    slot = [s for s, r in enumerate(nrows) for _ in range(r)]
    kvlen = [lens[s] - r + 1 + i for s, r in enumerate(nrows) for i in range(r)]
    row0 = [sum(nrows[:s]) for s in range(n)]
    monkeypatch.setattr(ops, "sm_count", ctas)
    check_attention(ops, 4, L, nq, page, slot, kvlen, table, cache, bf(g, len(slot), nq, L + R), (L + R) ** -0.5,
                    (i32(list(range(n))), i32(row0), i32(nrows), max(nrows)))
