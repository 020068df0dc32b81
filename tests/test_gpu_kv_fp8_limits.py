"""The 8-bit cache on the GPU, at the limits of what its operators take."""
import pytest
import torch

from arctic_platform_b200.ops import _lib, kv_fp8
from arctic_platform_b200.utils import checked
from tests.test_gpu_kv_fp8 import BF16, FP16, _attend, _close, _filled, _plan, _want

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("D", [64, 128])
def test_a_position_behind_the_tables_is_left_out_and_reported(D):
    B, Hq, H = 5, 4, 2
    g = _gen(D)
    sums = torch.randn((B, (Hq + 2 * H) * D), device="cuda", generator=g)
    w = torch.randn(D, device="cuda", generator=g).bfloat16()
    angle = torch.randn((9, D // 2), device="cuda", generator=g)
    rope = angle.cos().contiguous(), angle.sin().contiguous()
    slots = torch.arange(B, device="cuda", dtype=torch.int32)
    pos = torch.tensor([3, 9, 8, -1, 0], device="cuda", dtype=torch.int32)
    good = torch.tensor([True, False, True, False, True], device="cuda")
    want = kv_fp8.Fp8KVCache.zeros(1, H, D)
    q_want = kv_fp8.norm_rope_write(sums.clone(), w, w, rope, pos.clamp(0, 8), torch.where(good, slots, -1), want, Hq, 1e-6)
    checked.force(False)
    try:
        got, acc = kv_fp8.Fp8KVCache.zeros(1, H, D), sums.clone()
        q = kv_fp8.norm_rope_write(acc, w, w, rope, pos, slots, got, Hq, 1e-6)
        with pytest.raises(_lib.KernelError, match="203"):
            _lib.check_status("step")
        checked.force(True)
        with pytest.raises(checked.TableError, match="positions"):
            kv_fp8.norm_rope_write(sums.clone(), w, w, rope, pos, slots, got, Hq, 1e-6)
    finally:
        checked.force(None)
    assert torch.equal(got.data, want.data) and torch.equal(q[good], q_want[good]) and not q[~good].any() and not acc.any()


def test_weights_on_the_host_are_refused():
    sums = torch.zeros((1, 4 * 64), device="cuda")
    w = torch.ones(64).bfloat16()
    rope = torch.ones((2, 32), device="cuda"), torch.zeros((2, 32), device="cuda")
    at = torch.zeros(1, device="cuda", dtype=torch.int32)
    for q_norm, k_norm in ((w, None), (None, w), (w.cuda(), w)):
        with pytest.raises(ValueError, match="_norm lives on cpu"):
            kv_fp8.norm_rope_write(sums, q_norm, k_norm, rope, at, at, kv_fp8.Fp8KVCache.zeros(1, 1, 64), 2, 1e-6)


def test_a_table_far_wider_than_its_sequences():
    """More places in the table than shares of pages count; the sequences' lengths decide, not the table's width."""
    H, Hq, D, B, wide = 8, 32, 128, 16, 1 << 23
    cache, table, n, _ = _filled([300], H, D)
    table = torch.cat([table, torch.full((1, wide - table.shape[1]), -1, device="cuda", dtype=torch.int32)], 1).expand(B, -1)
    n = torch.arange(1, 301, 19, device="cuda", dtype=torch.int32)
    assert len(n) == B and kv_fp8._fn("scratch")(B, 5000 // 16, Hq, H, D) > 0
    q = torch.randn((B, Hq, D), device="cuda", generator=_gen(1)).bfloat16()
    checked.force(False)
    try:
        _close(kv_fp8.decode_attention(q, cache, table, n, longest=5000), *_want(q, cache, table, n))
    finally:
        checked.force(None)
    _lib.check_status("decode")


def test_a_table_of_as_many_places_as_there_are_tokens_in_32_bits():
    cache, table, n, _ = _filled([300], 1, 64)
    wide = torch.cat([table[0], torch.full(((1 << 27) - table.shape[1],), -1, device="cuda", dtype=torch.int32)])[None]
    q = torch.randn((1, 4, 64), device="cuda", generator=_gen(1)).bfloat16()
    checked.force(False)
    try:
        for longest in (300, None):
            _close(kv_fp8.decode_attention(q, cache, wide, n, longest=longest), *_want(q, cache, table, n))
    finally:
        checked.force(None)
    _lib.check_status("decode")


@pytest.mark.parametrize("size", [(1e36, 1e-28), (1e-28, 1e36), (3e-37, 1e30)])
@pytest.mark.parametrize("form,new,D", [("few", 2, 128), ("one tile", 9, 64), ("one tile", 9, 128), ("ctas", 150, 64), ("ctas", 150, 128), ("pairs", 150, 128)])
def test_queries_and_keys_of_any_size(monkeypatch, form, new, D, size):
    """Far apart, with a scale that brings their products back.  Queries and keys round as any others do: the tolerance is the usual one."""
    H, R, n = 2, 4, 420
    cache, table, lengths, slots = _filled([n], H, D, seed=3)
    g = _gen(10)
    k, v = (torch.randn((n, H, D), device="cuda", generator=g) for _ in range(2))
    q = torch.randn((new, H * R, D), device="cuda", generator=g)
    scale = D ** -0.5 / (size[0] * size[1])
    q = (q * size[0]).bfloat16()
    kv_fp8.write(k * size[1], v, slots, cache)
    plan = _plan(monkeypatch, form, [new], [n], table, H * R, cache)
    k, v = kv_fp8.read(cache, slots, torch.float32)
    want, most = _attend(q, k, v, torch.arange(n - new, n, device="cuda"), scale)
    _close(kv_fp8.chunk_attention(q, cache, plan, scale), want, most, FP16 if form == "few" else BF16)
    _close(kv_fp8.decode_attention(q[-1:], cache, table, lengths, scale), want[-1:], most[-1:])
    _lib.check_status("chunk")


@pytest.mark.parametrize("form,new", [("few", 2), ("one tile", 9), ("ctas", 300), ("pairs", 300)])
def test_one_query_for_all_tokens(monkeypatch, form, new):
    H, Hq, D = 2, 8, 128
    cache, table, n, _ = _filled([400, 330], H, D)
    plan = _plan(monkeypatch, form, [new] * 2, [400, 330], table, Hq, cache)
    q = torch.randn((1, Hq, D), device="cuda", generator=_gen(2)).bfloat16().expand(2 * new, -1, -1)
    want = kv_fp8.chunk_attention(q.contiguous(), cache, plan)
    assert torch.equal(kv_fp8.chunk_attention(q, cache, plan), want)
    assert torch.equal(kv_fp8.decode_attention(q[:2], cache, table, n), kv_fp8.decode_attention(q[:2].contiguous(), cache, table, n))


@pytest.mark.parametrize("longest", [None, 20000])
@pytest.mark.parametrize("Hq,H,D", [(8, 2, 128), (12, 1, 128), (4, 4, 64)])
def test_sequences_that_are_not_active_give_zeros(Hq, H, D, longest):
    """Both kernels, captured: what is active is read when the call is replayed."""
    lengths = [40, 0, 700, 3000, 16, 1] * 3
    cache, table, n, _ = _filled(lengths, H, D, seed=2)
    q = torch.randn((len(lengths), Hq, D), device="cuda", generator=_gen(2)).bfloat16()
    active = torch.ones_like(n)
    kv_fp8.decode_attention(q, cache, table, n, longest=longest, active=active)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv_fp8.decode_attention(q, cache, table, n, longest=longest, active=active)
    for pattern in ([1] * 18, [0, 1, 1, 0, 1, 1] * 3, [-1] * 18, [0] * 9 + [1] * 9):
        active.copy_(torch.tensor(pattern))
        graph.replay()
        seen = n * (active > 0)
        _close(out, *_want(q, cache, table, seen))
        assert not out[seen == 0].any()
        assert torch.equal(kv_fp8.decode_attention(q, cache, table, n, longest=longest, active=active), out)
        assert torch.equal(kv_fp8.decode_attention(q, cache, table, seen, longest=longest), out)
    _lib.check_status("decode")


@pytest.mark.parametrize("T", [3, 5000])
def test_rows_beside_slots_behind_the_cache_are_written(T):
    """A row that cannot be written takes none with it: the others are in the cache as the plain expression has them."""
    H, D = 2, 64
    g = _gen(T)
    k, v = (torch.randn((T, H, D), device="cuda", generator=g) for _ in range(2))
    cache, host = kv_fp8.Fp8KVCache.zeros(T // 16 + 2, H, D), kv_fp8.Fp8KVCache.zeros(T // 16 + 2, H, D, device="cpu")
    slots = torch.randperm(cache.num_pages * 16, device="cuda", generator=g)[:T].to(torch.int32)
    bad = slots.clone()
    bad[1::3] = torch.tensor([cache.num_pages * 16, (1 << 31) - 1], device="cuda", dtype=torch.int32).repeat(T)[:len(bad[1::3])]
    there = torch.where(bad < cache.num_pages * 16, bad, -1)
    kv_fp8.write(k.cpu(), v.cpu(), there.cpu(), host)
    checked.force(False)
    try:
        kv_fp8.write(k, v, bad, cache)
        with pytest.raises(_lib.KernelError, match="203"):
            _lib.check_status("write")
        rows = kv_fp8.read(cache, bad, torch.float32)
        with pytest.raises(_lib.KernelError, match="203"):
            _lib.check_status("read")
    finally:
        checked.force(None)
    assert torch.equal(cache.data.cpu(), host.data) and host.data.any()
    for x, y in zip(rows, kv_fp8.read(host, there.cpu(), torch.float32)):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("check", [False, True])
def test_an_idle_row_may_have_any_position(check):
    B, Hq, H, D = 3, 4, 2, 64
    g = _gen(1)
    sums = torch.randn((B, (Hq + 2 * H) * D), device="cuda", generator=g)
    angle = torch.randn((9, D // 2), device="cuda", generator=g)
    rope = angle.cos().contiguous(), angle.sin().contiguous()
    slots = torch.tensor([4, -1, -1], device="cuda", dtype=torch.int32)
    caches = [kv_fp8.Fp8KVCache.zeros(1, H, D) for _ in range(2)]
    checked.force(check)
    try:
        a, b = (kv_fp8.norm_rope_write(sums.clone(), None, None, rope, torch.tensor(p, device="cuda", dtype=torch.int32), slots, c, Hq, 1e-6)
                for p, c in (([8, 9, -5], caches[0]), ([8, 0, 0], caches[1])))
    finally:
        checked.force(None)
    _lib.check_status("step")
    assert torch.equal(a[0], b[0]) and not a[1:].any() and torch.equal(caches[0].data, caches[1].data) and caches[0].data.any()
