"""Latent cache of the MLA models in 4 and 8 bits: what a row stands for, and the engine over it, on the CPU."""
import dataclasses
import warnings

import latent_rows as lr
import pytest
import torch

from ferrite_b200.config import EngineConfig, tiny_mla
from ferrite_b200.engine.engine import Engine
from ferrite_b200.engine.executor import Segment
from ferrite_b200.models.weights import init_weights
from ferrite_b200.ops import mla_cache
from ferrite_b200.ops.torch_ops import TorchOps


def groups(size):
    g = torch.Generator().manual_seed(size)
    r = lambda sc: torch.randn(size, generator=g, dtype=torch.float64) * sc
    one = torch.zeros(size, dtype=torch.float64)
    one[3] = -0.7
    return {"ordinary": r(1.0), "small": r(1e-5), "tiny": r(1e-8), "large": r(3e3), "beyond": r(1e6), "zero": one * 0, "one": one,
            "border": torch.tensor([7.0 if i == 0 else (i % 14 - 7) + 0.5 for i in range(size)], dtype=torch.float64),
            "e4m3 border": torch.tensor([448.0 if i == 0 else (8 + i % 8 + 0.5) * 2.0 ** (i % 5 - 10) for i in range(size)], dtype=torch.float64)}


@pytest.mark.parametrize("bits", [4, 8])
def test_values_of_a_group(bits):
    for name, y in groups(mla_cache.GROUP[bits]).items():
        got = mla_cache.quantised(y[None], bits)[0]
        want = torch.tensor([float(v) for v in lr.group_values(y, bits)], dtype=torch.float64)
        assert torch.equal(got, want), name
        assert torch.equal(got, got.to(torch.bfloat16).double()) and torch.equal(got, got.to(torch.float16).double()), name


@pytest.mark.parametrize("bits", [4, 8])
def test_a_value_that_is_no_number_takes_its_group(bits):
    y = torch.randn(2, 128, dtype=torch.float64)
    y[0, 5], y[1, 127] = float("nan"), float("-inf")
    got, size = mla_cache.quantised(y, bits), mla_cache.GROUP[bits]
    bad = torch.zeros(2, 128, dtype=torch.bool)
    bad[0, :size], bad[1, -size:] = True, True
    assert torch.equal(got.isnan(), bad)


def test_row_sizes():
    assert [mla_cache.row_bytes(512, 64, b) for b in (4, 8, 16)] == [416, 656, 1152]
    for L in (64, 128, 192, 256, 512):
        for b in (4, 8):
            assert mla_cache.row_bytes(L, 64, b) == lr.row_bytes(L, b)
    for L, R, b in ((80, 64, 4), (576, 64, 4), (512, 32, 8), (512, 64, 6)):
        assert not mla_cache.fits(L, R, b)
        with pytest.raises(ValueError):
            mla_cache.row_bytes(L, R, b)


@pytest.mark.parametrize("bits", [4, 8])
def test_prep_writes_and_rows_read_back(bits):
    """The CPU statement: values of the written rows, rows of segments and whole contexts in their places, zeros between."""
    L, nq, dn, page = 64, 3, 32, 8
    g = torch.Generator().manual_seed(bits)
    ops = TorchOps("cpu", torch.float32)
    T = 13
    kva, q, w = torch.randn(T, L + 64, generator=g), torch.randn(T, nq * (dn + 64), generator=g), torch.randn(L, generator=g) * 0.2
    inv = 1e4 ** (-torch.arange(32) / 32)
    slot, pos = torch.tensor([1] * 10 + [0] * 3), torch.tensor(list(range(3, 13)) + [0, 1, 2])
    table = torch.tensor([[2, 0], [3, 1]], dtype=torch.int32)
    cache = torch.zeros(4, page, L + 64)
    wuk = torch.randn(nq, L, dn, generator=g)
    got = ops.mla_prep(q, kva, w, wuk, inv, slot, pos, table, cache, page, nq, dn, L, 64, 1e-6, kv_bits=bits)
    values = torch.cat([mla_cache.quantised(lr.normed(kva, w, L, 1e-6), bits), lr.rotated(kva[:, L:], pos, inv)], 1).float()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    own = ops.mla_rows(cache, i32(1, 0), i32(3, 0), i32(10, 3), table, page, L, 64, T, kv_bits=bits)
    assert torch.equal(own[:, :L], values[:, :L]) and torch.allclose(own, values, atol=1e-6)
    whole = ops.mla_rows(cache, i32(1, 0), i32(3, 0), i32(10, 3), table, page, L, 64, 24, whole=True, kv_bits=bits)
    assert torch.equal(whole[3:13], own[:10]) and torch.equal(whole[16:19], own[10:]) and not whole[13:16].any() and not whole[19:].any()
    plain = ops.mla_prep(q, kva, w, wuk, inv, slot, pos, table, torch.zeros_like(cache), page, nq, dn, L, 64, 1e-6)
    assert torch.allclose(got, plain, atol=1e-5)


def steps(eng, prompt):
    out = [eng.forward([Segment(1, 0, prompt[:30], "all")])[0].clone()]
    return torch.cat(out + [eng.forward([Segment(1, 30 + i, [prompt[30 + i]], "last")])[0].clone() for i in range(10)])


def test_engine_keeps_latents_in_the_bits_asked_for():
    cfg = tiny_mla()
    w = init_weights(cfg, seed=0)
    prompt = torch.randint(0, cfg.vocab, (40,), generator=torch.Generator().manual_seed(1)).tolist()
    out, page = {}, {}
    for kv in ("bf16", "fp8", "int4"):
        eng = Engine(cfg, w, EngineConfig(n_slots=2, max_ctx=128, kv_dtype=kv), device="cpu")
        out[kv], page[kv] = steps(eng, prompt), eng.ex.kv_block_bytes()
        if kv != "bf16":                                # every cached latent is a fixed point of its format
            rows = eng.ex.k_cache[0].view(-1, 128)[:, :64].double()
            assert rows.any() and torch.equal(mla_cache.quantised(rows, mla_cache.BITS[kv]), rows)
    assert page["bf16"] > page["fp8"] > page["int4"] and page["int4"] == 64 * 176 * cfg.n_layers
    d = {kv: (out[kv] - out["bf16"]).norm() / out["bf16"].norm() for kv in out}
    assert 0 < d["fp8"] < d["int4"] < 0.5


def test_engine_says_where_latents_stay_as_they_are():
    cfg = tiny_mla(moe=False)
    with pytest.warns(UserWarning, match="latents"):
        eng = Engine(cfg, init_weights(cfg, seed=0), EngineConfig(n_slots=1, max_ctx=128, kv_dtype="int6"), device="cpu")
    assert eng.ex.latent_bits == 16
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        Engine(cfg, init_weights(cfg, seed=0), EngineConfig(n_slots=1, max_ctx=128, kv_dtype="int4"), device="cpu")


def test_widths_that_no_kernel_attends_stay_as_they_are():
    cfg = dataclasses.replace(tiny_mla(moe=False), kv_lora=192)
    assert mla_cache.fits(192, 64, 4) and 192 not in mla_cache.ATTENDED
    with pytest.warns(UserWarning, match="latents"):
        eng = Engine(cfg, init_weights(cfg, seed=0), EngineConfig(n_slots=1, max_ctx=128, kv_dtype="int4"), device="cpu")
    assert eng.ex.latent_bits == 16
