"""The 8-bit cache without a GPU: what a row becomes, the plain expressions of its operators, what is refused."""
import math

import numpy as np
import pytest
import torch

from arctic_platform_b200.ops import kv_fp8
from arctic_platform_b200.utils import checked


def _fill(H, D, tokens, seed=0, spare=2):
    g = torch.Generator().manual_seed(seed)
    pages = (tokens + 15) // 16
    cache = kv_fp8.Fp8KVCache.zeros(pages + spare, H, D, device="cpu")
    order = torch.randperm(pages + spare, generator=g)[:pages].to(torch.int32)
    t = torch.arange(tokens)
    slots = (order.long()[t // 16] * 16 + t % 16).to(torch.int32)
    k, v = torch.randn(tokens, H, D, generator=g), torch.randn(tokens, H, D, generator=g)
    kv_fp8.write(k, v, slots, cache)
    return cache, order, slots, k, v


def test_codes_are_the_nearest_and_exponents_the_least():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(400, 64, generator=g) * torch.exp(6 * torch.randn(400, 1, generator=g))
    codes, byte = kv_fp8.quantise_ref(x)
    e = byte.double() - 127
    most = x.abs().amax(-1).double()
    assert (most <= 448 * torch.exp2(e)).all() and (most > 448 * torch.exp2(e - 1)).all()
    grid = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    grid = grid[torch.isfinite(grid)]
    scaled = x.double() / torch.exp2(e)[:, None]
    best = (scaled[..., None] - grid).abs().amin(-1)
    got = codes.view(torch.float8_e4m3fn).double()
    assert torch.equal((scaled - got).abs(), best)


def test_values_are_bf16_numbers_half_a_step_off():
    cache, _, slots, k, v = _fill(3, 64, 100)
    for x, y in zip((k, v), kv_fp8.read(cache, slots, torch.float32)):
        assert torch.equal(y, y.bfloat16().float())
        step = x.abs().amax(-1, keepdim=True) / 224                      # at least 2^exponent
        assert ((x - y).abs() <= torch.maximum(x.abs() * 2.0 ** -4, step * 2.0 ** -10)).all()
    again = kv_fp8.read(cache, slots)
    other = kv_fp8.Fp8KVCache.zeros(cache.num_pages, 3, 64, device="cpu")
    kv_fp8.write(*again, slots, other)                                    # what has been rounded stays as it is
    assert torch.equal(kv_fp8.read(other, slots)[0], again[0]) and torch.equal(kv_fp8.read(other, slots)[1], again[1])


@pytest.mark.parametrize("row,exponent", [([0.0, 0.0], -100), ([448.0, 1.0], 0), ([448.5, 1.0], 1), ([449.0, -0.0], 1), ([math.inf, 2.0], 119),
                                          ([3.0e38, -1e30], 119), ([math.nan, 448.0], 0), ([1e-45, 0.0], -100), ([-7.0, 7.0], -6)])
def test_edges_of_a_row(row, exponent):
    x = torch.tensor(row).repeat(32)[None]
    codes, byte = kv_fp8.quantise_ref(x)
    assert int(byte) - 127 == exponent
    y = kv_fp8.values_ref(codes, byte)[0]
    assert torch.equal(torch.isnan(y), torch.isnan(x[0])) and not torch.isinf(y).any()
    if exponent == 119:
        assert float(y.max()) == 448 * 2.0 ** 119


def test_order_and_portions_of_writing_do_not_matter():
    cache, _, slots, k, v = _fill(2, 64, 50)
    other = kv_fp8.Fp8KVCache.zeros(cache.num_pages, 2, 64, device="cpu")
    for i in torch.randperm(50).split(7):
        kv_fp8.write(k[i], v[i], slots[i], other)
    assert torch.equal(cache.data, other.data)


def test_slots_below_zero_are_left_out():
    cache, _, slots, k, v = _fill(2, 64, 40)
    before = cache.data.clone()
    kv_fp8.write(k + 1, v + 1, torch.full_like(slots, -1), cache)
    assert torch.equal(cache.data, before)
    some = slots.clone()
    some[::3] = -5
    a, _ = kv_fp8.read(cache, some)
    b, _ = kv_fp8.read(cache, slots)
    assert not a[::3].any() and torch.equal(a[1::3], b[1::3])


def test_attention_of_chunks_is_that_of_single_tokens():
    H, R, D, n = 2, 3, 64, 45
    cache, order, slots, _, _ = _fill(H, D, n)
    q = torch.randn(n, H * R, D, generator=torch.Generator().manual_seed(4)).bfloat16()
    plan = kv_fp8.ChunkPlan.build([n], [n], [order], H * R, cache)
    whole = kv_fp8.chunk_attention(q, cache, plan)
    table = order[None].repeat(n, 1)
    single = kv_fp8.decode_attention(q, cache, table, torch.arange(1, n + 1, dtype=torch.int32))
    # the same sums in another order, each rounded once: two half steps, and 2^-15 of fp32 sums of 45 terms of size 1
    assert ((whole.float() - single.float()).abs() <= 2 * 2.0 ** -8 * single.float().abs() + 2.0 ** -15).all()
    k, v = kv_fp8.read(cache, slots, torch.float32)
    s = torch.einsum("hd,thd->ht", q[-1].float(), k.repeat_interleave(R, 1)) / 8
    o = torch.einsum("ht,thd->hd", torch.softmax(s, -1), v.repeat_interleave(R, 1))
    assert torch.allclose(whole[-1].float(), o, atol=2.0 ** -15, rtol=2.0 ** -8)


def test_rows_that_see_nothing_and_rows_behind_the_last():
    cache, order, _, _, _ = _fill(1, 64, 20)
    q = torch.randn(9, 2, 64).bfloat16()
    plan = kv_fp8.ChunkPlan.build([4, 0, 3], [2, 7, 0], [order, order, order], 2, cache)     # more new tokens than the cache holds
    out = torch.full_like(q, 5.0)
    got = kv_fp8.chunk_attention(q, cache, plan, out=out)
    assert got is out and not out[:2].any() and out[2:4].abs().min() > 0 and not out[4:7].any() and (out[7:] == 5).all()
    assert not kv_fp8.chunk_attention(q, cache, plan)[7:].any()
    assert not kv_fp8.decode_attention(q[:1], cache, order[None], torch.zeros(1, dtype=torch.int32)).any()


def _refusals():
    cache = kv_fp8.Fp8KVCache.zeros(4, 2, 64, device="cpu")
    layers = kv_fp8.Fp8KVCache.zeros(4, 2, 64, device="cpu", layers=3)
    k = torch.zeros(5, 2, 64)
    s = torch.arange(5, dtype=torch.int32)
    q = torch.zeros(3, 4, 64).bfloat16()
    table, n = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    plan = lambda **a: kv_fp8.ChunkPlan.build(**{**dict(new=[1], lengths=[17], pages=[[0, 1]], heads=4, cache=cache), **a})  # noqa: E731
    return {
        "head size": lambda: kv_fp8.Fp8KVCache.zeros(4, 2, 96, device="cpu"),
        "no pages": lambda: kv_fp8.Fp8KVCache.zeros(0, 2, 64, device="cpu"),
        "block size": lambda: kv_fp8.Fp8KVCache(torch.zeros(4, 2, 100, dtype=torch.uint8), 64),
        "type of the cache": lambda: kv_fp8.Fp8KVCache(torch.zeros(4, 2, 2080), 64),
        "cache in strides": lambda: kv_fp8.Fp8KVCache(torch.zeros(4, 4, 2080, dtype=torch.uint8)[:, ::2], 64),
        "several layers": lambda: kv_fp8.write(k, k, s, layers),
        "type of the rows": lambda: kv_fp8.write(k.half(), k.half(), s, cache),
        "two types": lambda: kv_fp8.write(k, k.bfloat16(), s, cache),
        "heads of the rows": lambda: kv_fp8.write(k[:, :1], k[:, :1], s, cache),
        "number of rows": lambda: kv_fp8.write(k[:4], k[:4], s, cache),
        "type of the slots": lambda: kv_fp8.write(k, k, s.long(), cache),
        "a slot behind the cache": lambda: kv_fp8.write(k, k, s + 60, cache),
        "reading behind the cache": lambda: kv_fp8.read(cache, s + 60),
        "type to read": lambda: kv_fp8.read(cache, s, torch.float16),
        "type of the queries": lambda: kv_fp8.decode_attention(q.float(), cache, table, n),
        "query heads": lambda: kv_fp8.decode_attention(q[:, :3], cache, table, n),
        "head size of the queries": lambda: kv_fp8.decode_attention(torch.zeros(3, 4, 128).bfloat16(), cache, table, n),
        "rows of the table": lambda: kv_fp8.decode_attention(q, cache, table[:2], n),
        "type of the lengths": lambda: kv_fp8.decode_attention(q, cache, table, n.long()),
        "columns in strides": lambda: kv_fp8.decode_attention(q, cache, torch.zeros(3, 4, dtype=torch.int32)[:, ::2], n),
        "output in strides": lambda: kv_fp8.decode_attention(q, cache, table, n, out=torch.zeros(3, 64, 4).bfloat16().transpose(1, 2)),
        "counts": lambda: plan(new=[1, 2]),
        "negative length": lambda: plan(lengths=[-1]),
        "too few pages": lambda: plan(pages=[[0]]),
        "a page behind the cache": lambda: plan(pages=[[0, 4]]),
        "a page below 0": lambda: plan(pages=[[-1, 0]]),
        "heads of the plan": lambda: plan(heads=3),
        "another plan's heads": lambda: kv_fp8.chunk_attention(q, cache, plan(heads=2)),
        "fewer rows than the plan": lambda: kv_fp8.chunk_attention(q[:0], cache, plan()),
    }


@pytest.mark.parametrize("what", sorted(_refusals()))
def test_refusals(what):
    with pytest.raises(ValueError):
        _refusals()[what]()


def test_pages_behind_a_sequence_are_not_looked_at():
    cache, order, _, _, _ = _fill(1, 64, 20)
    table = torch.tensor([[int(order[0]), int(order[1]), -7, 99]], dtype=torch.int32)
    q = torch.randn(1, 1, 64).bfloat16()
    want = kv_fp8.decode_attention(q, cache, table[:, :2].contiguous(), torch.tensor([20], dtype=torch.int32))
    assert torch.equal(kv_fp8.decode_attention(q, cache, table, torch.tensor([20], dtype=torch.int32)), want)
    kv_fp8.ChunkPlan.build([1], [20], table.numpy(), 1, cache)


def test_checked_mode_names_bad_tables():
    cache, order, slots, k, v = _fill(1, 64, 20)
    q = torch.randn(1, 1, 64).bfloat16()
    checked.force(True)
    try:
        with pytest.raises(checked.TableError, match="page_table"):
            kv_fp8.decode_attention(q, cache, torch.tensor([[0, 99]], dtype=torch.int32), torch.tensor([20], dtype=torch.int32))
        with pytest.raises(checked.TableError, match="slots"):
            kv_fp8.write(k, v, slots + 1000, cache)
        twice = slots.clone()
        twice[3] = twice[7]
        with pytest.raises(checked.TableError, match="slots"):
            kv_fp8.write(k, v, twice, cache)
        twice[3] = twice[7] = -1                                          # padding may repeat
        kv_fp8.write(k, v, twice, cache)
    finally:
        checked.force(None)


def test_plan_of_nothing():
    cache = kv_fp8.Fp8KVCache.zeros(4, 2, 64, device="cpu")
    plan = kv_fp8.ChunkPlan.build([], [], [], 4, cache)
    q = torch.randn(2, 4, 64).bfloat16()
    assert not kv_fp8.chunk_attention(q, cache, plan).any()
    assert kv_fp8.decode_attention(q[:0], cache, torch.zeros(0, 3, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)).shape == (0, 4, 64)
    kv_fp8.write(torch.zeros(0, 2, 64), torch.zeros(0, 2, 64), torch.zeros(0, dtype=torch.int32), cache)
    assert kv_fp8.read(cache, torch.zeros(0, dtype=torch.int32))[0].shape == (0, 2, 64)
    assert np.array_equal(plan.new, [])


def test_names_of_cache_types():
    from arctic_platform_b200.engine.sampler import kv_cache_in_fp8
    assert [kv_cache_in_fp8(n) for n in (None, "", "auto", "bfloat16", "fp8", "fp8_e4m3")] == [False] * 4 + [True] * 2
    with pytest.raises(ValueError):
        kv_cache_in_fp8("int8")


def test_engines_without_it_say_so(caplog):
    from arctic_platform_b200.engine.reference_sampler import ReferenceSampler
    from arctic_platform_b200.engine.sampler import SamplerEngine
    from arctic_platform_b200.engine.worker import EngineWorker
    assert EngineWorker._kv_cache_dtype(SamplerEngine, {"kv_cache_dtype": "fp8"}) == {"kv_cache_dtype": "fp8"}
    assert EngineWorker._kv_cache_dtype(ReferenceSampler, {"kv_cache_dtype": "auto"}) == {} and not caplog.records
    assert EngineWorker._kv_cache_dtype(ReferenceSampler, {"kv_cache_dtype": "fp8"}) == {} and "ReferenceSampler" in caplog.text
