"""The 8-bit cache on the GPU: rows against the plain expressions (equal to the last bit), attention against 64 bits.

Tolerance of attention.  Operands of the products are exact (every value of the cache is a bf16 number).  A weight is rounded once, by
half a step: of fp16 in decode attention, 2^-11 of it at most, of bf16 in that of chunks (7 bits behind the point, so half a step of
1.0 is 2^-8), so that the sum is off by that much of sum_j p_j |v_j| at most; fp32 sums of up to 4096 terms and base-2 exponentials of
arguments below 2^7 in size add at most 2^-12 of the same; the result is rounded once to bf16, by 2^-8 of itself at most."""
import math

import pytest
import torch

from arctic_platform_b200.ops import _lib, kv_fp8
from arctic_platform_b200.utils import checked

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _filled(lengths, H, D, seed=0, spare=3, spread=0.5, dtype=torch.bfloat16):
    """A cache with the tokens of some sequences on shuffled pages; table, lengths."""
    g = _gen(seed)
    need = [(n + 15) // 16 for n in lengths]
    pages = sum(need) + spare
    cache = kv_fp8.Fp8KVCache(torch.randint(0, 256, (pages, H, kv_fp8.block_bytes(D)), device="cuda", dtype=torch.uint8, generator=g), D)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(need + [1]) + 1), -1, device="cuda", dtype=torch.int32)
    at = 0
    slots = []
    for s, (n, m) in enumerate(zip(lengths, need)):
        table[s, :m] = order[at:at + m]
        at += m
        t = torch.arange(n, device="cuda")
        slots.append((table[s].long()[t // 16] * 16 + t % 16).to(torch.int32))
    slots = torch.cat(slots)
    x = [torch.randn((len(slots), H, D), device="cuda", generator=g) * torch.exp(spread * torch.randn((len(slots), H, 1), device="cuda", generator=g))
         for _ in range(2)]
    kv_fp8.write(x[0].to(dtype), x[1].to(dtype), slots, cache)
    return cache, table, torch.tensor(lengths, device="cuda", dtype=torch.int32), slots


def _attend(q, k, v, last, scale):
    """64 bits: output and sum of p |v|."""
    rep = q.shape[1] // k.shape[1]
    k, v = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    s = torch.einsum("ihd,thd->hit", q.double(), k) * scale
    s = s.masked_fill(torch.arange(k.shape[0], device=q.device) > last[:, None], -math.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    return torch.einsum("hit,thd->ihd", p, v), torch.einsum("hit,thd->ihd", p, v.abs())


FP16, BF16 = 2.0 ** -11, 2.0 ** -8         # half a step of a weight


def _close(got, want, size, weight=FP16):
    bound = (weight + 2.0 ** -12) * size + 2.0 ** -8 * want.abs() + 1e-30
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), float((off / bound).max())


def _want(q, cache, table, lengths, new=None, scale=None):
    outs, row = [], 0
    for s, n in enumerate(lengths.tolist()):
        m = 1 if new is None else new[s]
        t = torch.arange(n, device="cuda")
        k, v = kv_fp8.read(cache, (table[s].long()[t // 16] * 16 + t % 16).to(torch.int32), torch.float32)
        outs.append(_attend(q[row:row + m], k, v, torch.arange(n - m, n, device="cuda"), scale or q.shape[2] ** -0.5)
                    if n else (torch.zeros_like(q[row:row + m], dtype=torch.float64),) * 2)
        row += m
    return torch.cat([o for o, _ in outs]), torch.cat([z for _, z in outs])


# --------------------------------------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,H,D", [(1, 1, 64), (1, 8, 128), (7, 3, 64), (16, 2, 128), (333, 5, 128), (1001, 2, 64), (5000, 8, 128)])
def test_rows_are_those_of_the_plain_expression(T, H, D, dtype):
    g = _gen(T)
    x = torch.randn((2, T, H, D), device="cuda", generator=g) * torch.exp(8 * torch.randn((2, T, H, 1), device="cuda", generator=g))
    x[0, 0, 0, :6] = torch.tensor([0.0, -0.0, 1e-38, 448.0, 3e38, -5e-42], device="cuda")
    x[1, T // 2] = 0
    k, v = x.to(dtype)
    cache = kv_fp8.Fp8KVCache(torch.randint(0, 256, (T // 16 + 3, H, kv_fp8.block_bytes(D)), device="cuda", dtype=torch.uint8, generator=g), D)
    host = kv_fp8.Fp8KVCache(cache.data.cpu(), D)
    slots = torch.randperm(cache.num_pages * 16, device="cuda", generator=g)[:T].to(torch.int32)
    slots[T // 3::7] = -2
    kv_fp8.write(k, v, slots, cache)
    kv_fp8.write(k.cpu(), v.cpu(), slots.cpu(), host)
    assert torch.equal(cache.data.cpu(), host.data)               # rows that nothing was written to, too
    for to in (torch.bfloat16, torch.float32):
        for a, b in zip(kv_fp8.read(cache, slots, to), kv_fp8.read(host, slots.cpu(), to)):
            assert a.dtype == to and torch.equal(a.cpu().nan_to_num(7.0), b.nan_to_num(7.0))


def test_numbers_that_are_none_and_infinities():
    k = torch.ones((2, 1, 64), device="cuda")
    k[0, 0, 3] = math.nan
    k[1, 0, 5], k[1, 0, 6] = math.inf, -math.inf
    cache = kv_fp8.Fp8KVCache.zeros(1, 1, 64)
    slots = torch.tensor([4, 5], device="cuda", dtype=torch.int32)
    kv_fp8.write(k, k, slots, cache)
    y, _ = kv_fp8.read(cache, slots, torch.float32)
    assert torch.isnan(y[0, 0, 3]) and (y[0, 0, torch.arange(64) != 3] == 1).all()
    assert y[1, 0, 5] == 448 * 2.0 ** 119 and y[1, 0, 6] == -448 * 2.0 ** 119 and y[1, 0, 0] == 0


@pytest.mark.parametrize("view", ["columns", "heads", "odd start", "transposed", "expanded"])
def test_rows_in_strides(view):
    g = _gen(5)
    T, H, D = 37, 4, 128
    if view == "columns":
        k = torch.randn((T, 3 * H * D), device="cuda", generator=g).bfloat16()[:, H * D:2 * H * D].unflatten(1, (H, D))
    elif view == "heads":
        k = torch.randn((T, 2 * H, D), device="cuda", generator=g).bfloat16()[:, ::2]
    elif view == "odd start":
        k = torch.randn(T * H * D + 3, device="cuda", generator=g).bfloat16()[3:].view(T, H, D)
    elif view == "transposed":
        k = torch.randn((H, D, T), device="cuda", generator=g).bfloat16().permute(2, 0, 1)
    else:
        k = torch.randn((T, 1, D), device="cuda", generator=g).bfloat16().expand(T, H, D)
    a, b = (kv_fp8.Fp8KVCache.zeros(3, H, D) for _ in range(2))
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    kv_fp8.write(k, -k, slots, a)
    kv_fp8.write(k.contiguous(), -k.contiguous(), slots, b)
    assert torch.equal(a.data, b.data)


def test_slots_behind_the_cache_are_left_out_and_reported():
    cache = kv_fp8.Fp8KVCache.zeros(2, 2, 64)
    k = torch.randn((3, 2, 64), device="cuda")
    slots = torch.tensor([1, 32, 1 << 30], device="cuda", dtype=torch.int32)
    kv_fp8.write(k, k, slots, cache)
    with pytest.raises(_lib.KernelError, match="203"):
        _lib.check_status("write")
    assert not kv_fp8.read(cache, slots)[0][1:].any()
    with pytest.raises(_lib.KernelError, match="203"):
        _lib.check_status("read")
    assert torch.equal(kv_fp8.read(cache, slots[:1])[0], kv_fp8.read(cache, slots[:1].clone())[0])
    _lib.check_status("read")


# --------------------------------------------------------------------------------------------- single tokens
@pytest.mark.parametrize("Hq,H,D", [(1, 1, 64), (4, 2, 64), (32, 8, 128), (5, 1, 128), (14, 2, 64), (32, 4, 128), (16, 1, 128), (40, 2, 64),
                                    (17, 1, 128), (64, 8, 128), (3, 3, 128)])
@pytest.mark.parametrize("lengths", [[1], [16], [17, 0, 33], [1, 2, 15, 16, 31, 32, 48, 129, 500, 0, 1023]])
def test_decode(Hq, H, D, lengths):
    cache, table, n, _ = _filled(lengths, H, D, seed=Hq)
    q = torch.randn((len(lengths), Hq, D), device="cuda", generator=_gen(1)).bfloat16()
    got = kv_fp8.decode_attention(q, cache, table, n)
    _close(got, *_want(q, cache, table, n))
    assert not got[n == 0].any()
    _lib.check_status("decode")


@pytest.mark.parametrize("B,length,Hq,H,D", [(1, 40000, 16, 1, 128), (1, 9000, 32, 8, 128), (2, 33333, 32, 4, 128), (130, 700, 32, 8, 128),
                                             (300, 90, 16, 8, 64), (1, 70000, 4, 2, 64), (3, 5000, 20, 1, 128)])
def test_decode_sizes(B, length, Hq, H, D):
    lengths = [max(0, length - (i * 7919) % length) for i in range(B)]
    cache, table, n, _ = _filled(lengths, H, D, seed=B)
    q = torch.randn((B, Hq, D), device="cuda", generator=_gen(2)).bfloat16()
    _close(kv_fp8.decode_attention(q, cache, table, n), *_want(q, cache, table, n))


@pytest.mark.parametrize("longest", [None, 0, 20000, 1 << 30])
@pytest.mark.parametrize("Hq,H,D", [(8, 2, 128), (12, 1, 128), (4, 4, 64)])
def test_decode_of_one_long_among_short_ones(Hq, H, D, longest):
    """Whatever the hint about lengths says: shares of pages that many short sequences fill, and one sequence over many shares."""
    lengths = [1, 0, 17, 5] * 20 + [0, 0, 20000, 3] + [40] * 9 + [0]
    cache, table, n, _ = _filled(lengths, H, D, seed=2)
    wide = torch.cat([table, torch.full((len(lengths), 900), -3, device="cuda", dtype=torch.int32)], 1)
    q = torch.randn((len(lengths), Hq, D), device="cuda", generator=_gen(2)).bfloat16()
    want = _want(q, cache, table, n)
    out = torch.full_like(q, 7.0)
    for t in (table, wide):
        _close(kv_fp8.decode_attention(q, cache, t, n, out=out, longest=longest), *want)
    assert not out[n == 0].any()
    again = kv_fp8.decode_attention(q, cache, wide, n, longest=longest)
    assert torch.equal(again, out)
    _lib.check_status("decode")


@pytest.mark.parametrize("case", ["large", "small", "values of unlike size", "one huge value nobody sees", "steep", "negative scale", "zero scale"])
def test_decode_numbers(case):
    H, D, n = 2, 128, 300
    cache, table, lengths, slots = _filled([n], H, D, seed=3)
    g = _gen(9)
    k, v = (torch.randn((n, H, D), device="cuda", generator=g) for _ in range(2))
    q = torch.randn((1, 8, D), device="cuda", generator=g)
    scale = D ** -0.5
    if case == "large":
        k, v, q = k * 1e15, v * 1e30, q * 1e-15
    elif case == "small":
        k, v, q = k * 1e-12, v * 1e-22, q * 1e12
    elif case == "values of unlike size":
        v = v * torch.exp(12 * torch.randn((n, H, 1), device="cuda", generator=g))
    elif case == "one huge value nobody sees":
        q[:, :, 0], k[:, :, 0] = 30.0, 0.0
        k[77, :, 0] = -400.0                    # its weight is 2^-1500
        v[77] = 1e30
    elif case == "steep":
        q = q * 60
    elif case == "negative scale":
        scale = -0.3
    else:
        scale = 0.0
    kv_fp8.write(k, v, slots, cache)
    q = q.bfloat16()
    got = kv_fp8.decode_attention(q, cache, table, lengths, scale)
    k, v = kv_fp8.read(cache, slots, torch.float32)
    want, size = _attend(q, k, v, lengths - 1, scale)
    if case in ("steep", "values of unlike size"):
        # scores of up to 2^9 are sums in fp32 and go into the exponential with a 2^-24 of their size: weights are off by 2^-13 more
        size = size * 1.25               # (2^-11 + 2^-12) * 1.25 > 2^-11 + 2^-12 + 2^-13
    _close(got, want, size)
    plan = kv_fp8.ChunkPlan.build([1], [n], table.cpu().numpy(), 8, cache)
    _close(kv_fp8.chunk_attention(q, cache, plan, scale), want, size, BF16)


def test_no_number_behind_the_last_token_is_seen():
    """Bytes that nothing was written to, in the last page and in others, are no numbers."""
    H, D = 2, 128
    cache, table, n, slots = _filled([21, 5], H, D, seed=4)
    want = kv_fp8.decode_attention(torch.ones((2, 4, D), device="cuda").bfloat16(), cache, table, n)
    k, v = kv_fp8.read(cache, slots, torch.float32)
    cache.data.fill_(0x7F)
    kv_fp8.write(k, v, slots, cache)
    got = kv_fp8.decode_attention(torch.ones((2, 4, D), device="cuda").bfloat16(), cache, table, n)
    assert torch.equal(got, want)
    plan = kv_fp8.ChunkPlan.build([3, 5], [21, 5], table.cpu().numpy(), 4, cache)
    q = torch.ones((8, 4, D), device="cuda").bfloat16()
    _close(kv_fp8.chunk_attention(q, cache, plan), *_want(q, cache, table, n, [3, 5]), BF16)


def test_a_key_that_is_no_number_reaches_its_sequence_and_head_alone():
    H, D = 2, 64
    cache, table, n, slots = _filled([40, 40], H, D, seed=5)
    k, v = kv_fp8.read(cache, slots, torch.float32)
    k[10, 1, 3] = math.nan
    kv_fp8.write(k, v, slots, cache)
    q = torch.randn((2, 4, D), device="cuda", generator=_gen(1)).bfloat16()
    got = kv_fp8.decode_attention(q, cache, table, n)
    assert torch.isnan(got[0, 2:]).all() and torch.isfinite(got[0, :2]).all() and torch.isfinite(got[1]).all()


def test_bad_pages_are_left_out_and_reported():
    H, D = 2, 128
    cache, table, n, _ = _filled([64, 33], H, D, seed=6)
    q = torch.randn((2, 4, D), device="cuda", generator=_gen(1)).bfloat16()
    bad = table.clone()
    bad[0, 1], bad[1, 2] = cache.num_pages, -1
    checked.force(False)
    try:
        got = kv_fp8.decode_attention(q, cache, bad, n)
        with pytest.raises(_lib.KernelError, match="203"):
            _lib.check_status("decode")
        assert torch.isfinite(got).all()
        got = kv_fp8.decode_attention(q, cache, table[:, :2].contiguous(), n)     # longer than the table is wide
        with pytest.raises(_lib.KernelError, match="203"):
            _lib.check_status("decode")
        _close(got, *_want(q, cache, table, torch.tensor([32, 32], device="cuda")))
    finally:
        checked.force(None)
    with pytest.raises(ValueError):
        kv_fp8.ChunkPlan.build([1, 1], [64, 33], bad.cpu().numpy(), 4, cache)


def test_queries_tables_and_outputs_in_strides():
    H, D, lengths = 2, 128, [50, 17, 0, 90]
    cache, table, n, _ = _filled(lengths, H, D, seed=7)
    wide = torch.randn((4, 3 * 8 * D + 8), device="cuda", generator=_gen(1)).bfloat16()
    q = wide[:, 8 * D:16 * D].unflatten(1, (8, D))
    want = kv_fp8.decode_attention(q.contiguous(), cache, table, n)
    big = torch.full((4, table.shape[1] + 5), -9, device="cuda", dtype=torch.int32)
    big[:, 2:2 + table.shape[1]] = table
    out = torch.full((4, 24, D), 5.0, device="cuda").bfloat16()
    got = kv_fp8.decode_attention(q, cache, big[:, 2:2 + table.shape[1]], n, out=out[:, 8:16])
    assert torch.equal(got, want) and (out[:, :8] == 5).all() and (out[:, 16:] == 5).all()
    odd = torch.empty(4 * 8 * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(4, 8, D)
    odd.copy_(q)
    assert torch.equal(kv_fp8.decode_attention(odd, cache, table, n), want)
    odd_out = torch.empty(4 * 8 * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(4, 8, D)
    kv_fp8.decode_attention(q, cache, table, n, out=odd_out)
    assert torch.equal(odd_out, want)


# --------------------------------------------------------------------------------------------- chunks
@pytest.mark.parametrize("Hq,H,D", [(1, 1, 64), (4, 2, 64), (32, 8, 128), (5, 1, 128), (14, 2, 64), (16, 1, 128), (64, 8, 128), (3, 3, 128), (40, 1, 64)])
@pytest.mark.parametrize("new,lengths", [([1], [1]), ([5], [5]), ([2], [130]), ([3, 0, 17, 1], [200, 40, 17, 0]), ([129, 64, 1], [129, 300, 257]),
                                         ([5] * 9, [7, 5, 100, 33, 16, 17, 640, 5, 21]), ([4, 300], [2, 290])])
def test_chunks(Hq, H, D, new, lengths):
    cache, table, n, _ = _filled(lengths, H, D, seed=Hq)
    q = torch.randn((sum(new), Hq, D), device="cuda", generator=_gen(3)).bfloat16()
    plan = kv_fp8.ChunkPlan.build(new, lengths, table.cpu().numpy(), Hq, cache)
    _close(kv_fp8.chunk_attention(q, cache, plan), *_want(q, cache, table, n, new), BF16)
    _lib.check_status("chunk")


@pytest.mark.parametrize("new,lengths,Hq,H,D", [([2000], [2000], 32, 8, 128), ([700, 1], [5000, 9000], 16, 8, 128), ([16], [30000], 32, 4, 128),
                                                ([1500, 33, 900], [1500, 700, 1700], 14, 2, 64), ([1] * 40, [901] * 40, 8, 1, 128)])
def test_chunk_sizes(new, lengths, Hq, H, D):
    cache, table, n, _ = _filled(lengths, H, D, seed=1)
    q = torch.randn((sum(new), Hq, D), device="cuda", generator=_gen(3)).bfloat16()
    plan = kv_fp8.ChunkPlan.build(new, lengths, table.cpu().numpy(), Hq, cache)
    _close(kv_fp8.chunk_attention(q, cache, plan), *_want(q, cache, table, n, new), BF16)


def test_padding_rows_of_a_chunk_are_left():
    cache, table, n, _ = _filled([30, 50], 2, 128, seed=2)
    q = torch.randn((300, 8, 128), device="cuda", generator=_gen(3)).bfloat16()
    plan = kv_fp8.ChunkPlan.build([30, 7], [30, 50], table.cpu().numpy(), 8, cache)
    want, size = _want(q[:37], cache, table, n, [30, 7])
    out = torch.full_like(q, 3.0)
    kv_fp8.chunk_attention(q, cache, plan, out=out)
    _close(out[:37], want, size, BF16)
    assert (out[37:] == 3).all()
    assert not kv_fp8.chunk_attention(q, cache, plan)[37:].any()
    wide = torch.full((300, 24, 128), 3.0, device="cuda").bfloat16()
    kv_fp8.chunk_attention(q, cache, plan, out=wide[:, 8:16])
    assert torch.equal(wide[:37, 8:16], out[:37]) and (wide[:, :8] == 3).all() and (wide[37:] == 3).all()


def _plan(monkeypatch, form, new, lengths, table, Hq, cache):
    """With items taken in this form (csrc/runtime_kv8.cpp), whichever is sooner done; "few": without items."""
    work, number = kv_fp8._work, {"ctas": 0, "one tile": 1, "pairs": 2, "few": None}[form]
    monkeypatch.setattr(kv_fp8, "_work", lambda *a: work(*a, form=number))
    monkeypatch.setattr(kv_fp8, "_few", lambda *a: form == "few")
    plan = kv_fp8.ChunkPlan.build(new, lengths, table.cpu().numpy(), Hq, cache)
    assert (plan.work is None) if form == "few" else plan.work.form == number
    return plan


@pytest.mark.parametrize("form", ["ctas", "pairs"])
@pytest.mark.parametrize("new,lengths,Hq,H", [([512], [5000], 32, 8), ([700, 1, 33], [700, 9000, 40], 16, 8), ([1300] * 3, [1300, 1290, 2000], 5, 1),
                                              ([150, 20], [150, 3000], 130, 1), ([65] * 90, [65 + 17 * i for i in range(90)], 64, 4)])
def test_long_chunks_by_ctas_and_by_pairs(monkeypatch, form, new, lengths, Hq, H):
    """Rows that see nothing (a length below the new tokens), tiles that no token fills, more heads than a tile has rows."""
    cache, table, n, _ = _filled(lengths, H, 128, seed=4)
    q = torch.randn((sum(new), Hq, 128), device="cuda", generator=_gen(5)).bfloat16()
    plan = _plan(monkeypatch, form, new, lengths, table, Hq, cache)
    _close(kv_fp8.chunk_attention(q, cache, plan), *_want(q, cache, table, n, new), BF16)
    _lib.check_status("chunk")


@pytest.mark.parametrize("form,new,D", [("few", 4, 64), ("few", 2, 128), ("one tile", 9, 64), ("one tile", 9, 128), ("ctas", 500, 64), ("ctas", 1500, 128), ("pairs", 1500, 128)])
def test_scores_that_grow_by_leaps(monkeypatch, form, new, D):
    """What a chunk's weights are relative to moves only when they pass 2^40: here the scores leap along the sequence, by little and by a
    lot, at the borders of blocks, inside of them and from one half of a block to the next, up and down again, and by head."""
    length, H, R = 2100, 2, 4
    g = _gen(6)
    base = torch.randn((H, D), device="cuda", generator=g)
    base /= base.square().sum(-1, keepdim=True).sqrt()
    height = torch.zeros(length, device="cuda")
    for at, to in ((0, 1.0), (40, 20.0), (100, 45.0), (128, 60.0), (200, 130.0), (256, 125.0), (320, 250.0), (600, 0.0), (1024, 290.0), (1100, -300.0),
                   (1536, 400.0), (2064, 560.0)):
        height[at:] = to
    k = base * height[:, None, None] + 0.3 * torch.randn((length, H, D), device="cuda", generator=g)
    v = torch.randn((length, H, D), device="cuda", generator=g) * torch.exp(torch.randn((length, H, 1), device="cuda", generator=g))
    cache = kv_fp8.Fp8KVCache.zeros((length + 15) // 16, H, D)
    table = torch.randperm(cache.num_pages, device="cuda", generator=g).to(torch.int32)[None]
    t = torch.arange(length, device="cuda")
    kv_fp8.write(k, v, (table[0].long()[t // 16] * 16 + t % 16).to(torch.int32), cache)
    q = (base.repeat_interleave(R, 0) * torch.linspace(-0.5, 1.0, H * R, device="cuda")[:, None] * D ** 0.5 * 0.7
         + 0.2 * torch.randn((new, H * R, D), device="cuda", generator=g)).bfloat16()
    n = torch.tensor([length], device="cuda", dtype=torch.int32)
    plan = _plan(monkeypatch, form, [new], [length], table, H * R, cache)
    want, size = _want(q, cache, table, n, [new])
    # scores of up to 400: eight sums in fp32 that a product of 16 terms each is added to, off by 2^-23 of it at most, leave weights off by
    # 8 * 2^-23 * 400 = 2^-11.3 more, and their sum likewise; (2^-8 + 2^-12) * 0.25 is above 2 * 2^-11.3 + 2^-14
    _close(kv_fp8.chunk_attention(q, cache, plan), want, size * 1.25, BF16)
    _lib.check_status("chunk")


@pytest.mark.parametrize("case", ["large", "small", "values of unlike size", "one huge value nobody sees", "steep", "negative scale", "zero scale",
                                  "nothing but one token"])
@pytest.mark.parametrize("form,new,D", [("few", 2, 128), ("one tile", 9, 64), ("one tile", 9, 128), ("ctas", 150, 64), ("ctas", 150, 128), ("pairs", 150, 128)])
def test_numbers_of_chunks(monkeypatch, form, new, D, case):
    H, R, n = 2, 4, 420
    cache, table, lengths, slots = _filled([n], H, D, seed=3)
    g = _gen(10)
    k, v = (torch.randn((n, H, D), device="cuda", generator=g) for _ in range(2))
    q = torch.randn((new, H * R, D), device="cuda", generator=g)
    scale = D ** -0.5
    if case == "large":
        k, v, q = k * 1e15, v * 1e30, q * 1e-15
    elif case == "small":
        k, v, q = k * 1e-12, v * 1e-22, q * 1e12
    elif case == "values of unlike size":
        v = v * torch.exp(12 * torch.randn((n, H, 1), device="cuda", generator=g))
    elif case == "one huge value nobody sees":
        q[:, :, 0], k[:, :, 0] = 30.0, 0.0
        k[77, :, 0] = -400.0
        v[77] = 1e20                            # 2^66, 2^67 of the others
    elif case == "steep":
        q = q * 40
    elif case == "negative scale":
        scale = -0.3
    elif case == "zero scale":
        scale = 0.0
    else:
        k, v = k * 0, v * 0
        v[5] = 1.0
    kv_fp8.write(k, v, slots, cache)
    q = q.bfloat16()
    plan = _plan(monkeypatch, form, [new], [n], table, H * R, cache)
    k, v = kv_fp8.read(cache, slots, torch.float32)
    want, size = _attend(q, k, v, torch.arange(n - new, n, device="cuda"), scale)
    if case in ("steep", "values of unlike size"):
        size = size * 1.25                     # scores of up to 400, as below
    _close(kv_fp8.chunk_attention(q, cache, plan, scale), want, size, FP16 if form == "few" else BF16)


@pytest.mark.parametrize("form,new,D", [("few", 2, 128), ("one tile", 9, 64), ("one tile", 9, 128), ("ctas", 150, 64), ("ctas", 150, 128), ("pairs", 150, 128)])
def test_numbers_that_are_none_in_a_chunk(monkeypatch, form, new, D):
    """A key that is none reaches the rows that see it, of its sequence and head; a value its column of them at least."""
    H, R = 2, 4
    lengths = [400, 300]
    cache, table, n, slots = _filled(lengths, H, D, seed=5)
    q = torch.randn((2 * new, H * R, D), device="cuda", generator=_gen(1)).bfloat16()
    plan = _plan(monkeypatch, form, [new] * 2, lengths, table, H * R, cache)
    k, v = kv_fp8.read(cache, slots, torch.float32)
    kv_fp8.write(k, v, slots, cache)                # a row whose largest was rounded down may get the next exponent, and the same numbers
    want = kv_fp8.chunk_attention(q, cache, plan)
    for token, column in ((10, 3), (200, D - 1), (400 - new + new // 2, 17), (399, 0)):
        bad = k.clone()
        bad[token, 1, column] = -math.nan
        kv_fp8.write(bad, v, slots, cache)
        got = kv_fp8.chunk_attention(q, cache, plan)
        sees = torch.arange(400 - new, 400, device="cuda") >= token
        assert torch.isnan(got[:new, R:][sees]).all()
        if not sees.all():             # the others may share a warp with rows that see it, and take another reference
            exact, size = _attend(q[:new], k[:400], v[:400], torch.arange(400 - new, 400, device="cuda"), D ** -0.5)
            _close(got[:new, R:][~sees], exact[:, R:][~sees], size[:, R:][~sees], FP16 if form == "few" else BF16)
        got[:new, R:] = want[:new, R:]
        assert torch.equal(got, want)
        bad = v.clone()
        bad[token, 1, column] = math.nan
        kv_fp8.write(k, bad, slots, cache)
        got = kv_fp8.chunk_attention(q, cache, plan)
        assert torch.isnan(got[:new, R:, column][sees]).all()
        got[:new, R:, column] = want[:new, R:, column]
        assert torch.equal(got, want)
    cache.data[int(table[0, 0]), 1, 3 * D] = 0xFF            # as other writers have them
    assert torch.isnan(kv_fp8.chunk_attention(q, cache, plan)[:new, R:]).all()


@pytest.mark.parametrize("Hq,H,D,new", [(8, 2, 64, 2), (32, 8, 128, 2), (32, 8, 128, 4), (3, 3, 128, 8), (5, 1, 128, 3), (16, 1, 64, 1), (7, 1, 128, 1),
                                        (12, 4, 64, 5)])
@pytest.mark.parametrize("lengths", [[1], [40, 0, 129, 3, 16, 17], [9000, 31, 2], [300 + 7 * i for i in range(70)]])
def test_few_tokens_of_each_sequence(monkeypatch, Hq, H, D, new, lengths):
    """Causal among themselves, with sequences that bring none, that bring less than others, or more than they have."""
    cache, table, n, _ = _filled(lengths, H, D, seed=Hq)
    news = [new if i % 3 != 2 else i % 2 * (new - 1) for i in range(len(lengths))]
    q = torch.randn((sum(news) + 3, Hq, D), device="cuda", generator=_gen(5)).bfloat16()
    plan = _plan(monkeypatch, "few", news, lengths, table, Hq, cache)
    out = torch.full_like(q, 3.0)
    kv_fp8.chunk_attention(q, cache, plan, out=out)
    _close(out[:-3], *_want(q[:-3], cache, table, n, news))
    assert (out[-3:] == 3).all()
    _lib.check_status("few")


@pytest.mark.parametrize("Hq,H,D,new", [(130, 1, 64, 2), (200, 1, 128, 3), (256, 2, 128, 1), (384, 1, 64, 40)])
def test_more_heads_than_a_tile_has_rows(Hq, H, D, new):
    lengths = [700, 33]
    cache, table, n, _ = _filled(lengths, H, D, seed=7)
    q = torch.randn((2 * new, Hq, D), device="cuda", generator=_gen(8)).bfloat16()
    plan = kv_fp8.ChunkPlan.build([new] * 2, lengths, table.cpu().numpy(), Hq, cache)
    _close(kv_fp8.chunk_attention(q, cache, plan), *_want(q, cache, table, n, [new] * 2), BF16)
    q = q[:2]
    _close(kv_fp8.decode_attention(q, cache, table, n), *_want(q, cache, table, n))


# --------------------------------------------------------------------------------------------- together
def test_a_sequence_step_by_step():
    """A prompt in chunks, then token after token: written, attended to, read back."""
    H, R, D, total = 2, 4, 128, 90
    g = _gen(8)
    q, k, v = (torch.randn((total, h, D), device="cuda", generator=g).bfloat16() for h in (H * R, H, H))
    cache = kv_fp8.Fp8KVCache.zeros(9, H, D, layers=2)
    layer = cache.layer(1)
    pages = torch.tensor([[7, 2, 5, 0, 8, 1]], device="cuda", dtype=torch.int32)
    t = torch.arange(total, device="cuda")
    slots = (pages[0].long()[t // 16] * 16 + t % 16).to(torch.int32)
    outs, at = [], 0
    for m in (33, 20, 7):
        kv_fp8.write(k[at:at + m], v[at:at + m], slots[at:at + m], layer)
        plan = kv_fp8.ChunkPlan.build([m], [at + m], pages.cpu().numpy(), H * R, layer)
        outs.append(kv_fp8.chunk_attention(q[at:at + m], layer, plan))
        at += m
    while at < total:
        kv_fp8.write(k[at:at + 1], v[at:at + 1], slots[at:at + 1], layer)
        outs.append(kv_fp8.decode_attention(q[at:at + 1], layer, pages, torch.tensor([at + 1], device="cuda", dtype=torch.int32)))
        at += 1
    kk, vv = kv_fp8.read(layer, slots, torch.float32)
    _close(torch.cat(outs), *_attend(q, kk, vv, t, D ** -0.5), BF16)
    assert not cache.data[0].any()


@pytest.mark.parametrize("what", ["decode", "long decode", "chunk", "split chunk"])
def test_two_graphs_and_two_streams(what):
    """Captured calls read their lengths at replay, do not share scratch, and give the bits of an eager call."""
    H, Hq, D = 2, 8, 128
    lengths = [20000, 3] if what in ("long decode", "split chunk") else [300, 65, 17]
    cache, table, n, _ = _filled(lengths, H, D, seed=9)
    new = [4] * len(lengths) if "chunk" in what else [1] * len(lengths)
    plan = kv_fp8.ChunkPlan.build(new, lengths, table.cpu().numpy(), Hq, cache)
    qs = [torch.randn((sum(new), Hq, D), device="cuda", generator=_gen(i)).bfloat16() for i in range(2)]
    call = (lambda q: kv_fp8.chunk_attention(q, cache, plan)) if "chunk" in what else (lambda q: kv_fp8.decode_attention(q, cache, table, n))
    want = [call(q).clone() for q in qs]
    graphs, outs = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(q))
        graphs.append(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for o in outs:
            o.zero_()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    if "decode" in what:
        n[1] = 0
        graphs[0].replay()
        assert not outs[0][1].any() and torch.equal(outs[0][0], want[0][0])
    with torch.cuda.stream(side):
        again = [call(q) for q in qs]
    torch.cuda.synchronize()
    assert torch.equal(again[0][0], want[0][0])


@pytest.mark.parametrize("form,new,lengths", [("few", 2, [900, 65, 17]), ("one tile", 9, [9000, 65, 17]), ("ctas", 300, [9000, 600, 300]),
                                              ("pairs", 300, [9000, 600, 300]), ("pairs", 40, [40] * 30)])
def test_chunks_captured_and_on_two_streams(monkeypatch, form, new, lengths):
    """Every form, replayed beside another graph and beside itself on a second stream, gives the bits of an eager call; a cache of
    another layer takes the same plan."""
    H, Hq, D = 2, 8, 128
    cache, table, n, _ = _filled(lengths, H, D, seed=9)
    other = kv_fp8.Fp8KVCache(cache.data.clone(), D)
    plan = _plan(monkeypatch, form, [new] * len(lengths), lengths, table, Hq, cache)
    qs = [torch.randn((new * len(lengths), Hq, D), device="cuda", generator=_gen(i)).bfloat16() for i in range(2)]
    want = [kv_fp8.chunk_attention(q, cache, plan).clone() for q in qs]
    _close(want[0], *_want(qs[0], cache, table, n, [new] * len(lengths)), FP16 if form == "few" else BF16)
    graphs, outs = [], []
    for q, c in zip(qs, (cache, other)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kv_fp8.chunk_attention(q, c, plan))
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(3):
        for o in outs:
            o.zero_()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            again = kv_fp8.chunk_attention(qs[0], other, plan)
        more = kv_fp8.chunk_attention(qs[1], cache, plan)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(again, want[0]) and torch.equal(more, want[1])
    in_place = qs[0].clone()
    kv_fp8.chunk_attention(in_place, cache, plan, out=in_place)
    assert torch.equal(in_place, want[0])
    _lib.check_status("chunk")


@pytest.mark.parametrize("what", ["decode", "chunk"])
def test_scratch_is_kept_until_the_launch_is_made(monkeypatch, what):
    """Another thread that allocates on the same stream meanwhile gets other memory."""
    H, Hq, D, lengths = 2, 8, 128, [20000, 3]
    cache, table, n, _ = _filled(lengths, H, D, seed=9)
    q = torch.randn((8, Hq, D), device="cuda", generator=_gen(0)).bfloat16()
    plan = _plan(monkeypatch, "one tile", [4, 4], lengths, table, Hq, cache)
    assert plan.work.part_tiles
    call = (lambda: kv_fp8.decode_attention(q[:2], cache, table, n)) if what == "decode" else (lambda: kv_fp8.chunk_attention(q, cache, plan))
    want = call().clone()
    size = kv_fp8._fn("scratch")(2, table.shape[1], Hq, H, D) if what == "decode" else plan.work.part_tiles * 128 * (D + 2) * 4
    assert size
    fn, others = kv_fp8._fn(what), []

    def interrupted(*args):
        others.append(torch.empty(size, device="cuda", dtype=torch.uint8))
        assert others[-1].data_ptr() not in [getattr(a, "value", a) for a in args]
        return fn(*args)

    monkeypatch.setitem(kv_fp8._FN, what, interrupted)
    assert torch.equal(call(), want) and len(others) == 1


def test_offsets_behind_two_to_the_31():
    H, D = 8, 128
    pages = (1 << 31) // (H * kv_fp8.block_bytes(D)) + 50
    cache = kv_fp8.Fp8KVCache(torch.empty((pages, H, kv_fp8.block_bytes(D)), device="cuda", dtype=torch.uint8), D)
    table = torch.tensor([[pages - 1, 0, pages - 30]], device="cuda", dtype=torch.int32)
    t = torch.arange(40, device="cuda")
    slots = (table[0].long()[t // 16] * 16 + t % 16).to(torch.int32)
    g = _gen(1)
    k, v = (torch.randn((40, H, D), device="cuda", generator=g).bfloat16() for _ in range(2))
    kv_fp8.write(k, v, slots, cache)
    small = kv_fp8.Fp8KVCache.zeros(3, H, D)
    kv_fp8.write(k, v, t.to(torch.int32), small)
    assert torch.equal(kv_fp8.read(cache, slots)[1], kv_fp8.read(small, t.to(torch.int32))[1])
    q = torch.randn((1, 16, D), device="cuda", generator=g).bfloat16()
    n = torch.tensor([40], device="cuda", dtype=torch.int32)
    order = torch.arange(3, device="cuda", dtype=torch.int32)[None]
    assert torch.equal(kv_fp8.decode_attention(q, cache, table, n), kv_fp8.decode_attention(q, small, order, n))
    plans = [kv_fp8.ChunkPlan.build([1], [40], p.cpu().numpy(), 16, c) for p, c in ((table, cache), (order, small))]
    assert torch.equal(kv_fp8.chunk_attention(q, cache, plans[0]), kv_fp8.chunk_attention(q, small, plans[1]))
