"""Tokens drawn on a GPU from rows of logits with given random numbers, against the expression in 64 bits.

Tokens are equal: masses are whole multiples of 2^-45 there and 64-bit numbers here, so that only a uniform within 1e-9 of a border could
tell them apart.  Log-probabilities: the denominator is an fp32 sum of at most 50 elements a thread, 16 warps and 8 parts (each addition off
by 2^-24 of the sum: 5e-6) of approximate exponentials (2^-22, and 2^-23 of the exponent, on average below 13 nats: 2e-6), its logarithm and
the result rounded to fp32."""
import pytest
import torch

from arctic_platform_b200.ops import sampling

pytestmark = pytest.mark.gpu
ATOL, RTOL = 2e-5, 2.0 ** -22


def make(B, V, dtype=torch.float32, seed=0, spare=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = spread * torch.randn((B, V + spare), device="cuda", generator=g)
    ids = torch.randint(V, (B, min(40, V)), device="cuda", generator=g)
    z.scatter_reduce_(1, ids, 4 + 8 * torch.rand(ids.shape, device="cuda", generator=g), "amax")
    return z.to(dtype)[:, :V], torch.rand(B, device="cuda", generator=g)


def same(z, u, *settings, out=None):
    got = sampling.sample(z, u, *settings, out=out)
    want = sampling.sample_ref(z, u, *settings)
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.float32
    torch.testing.assert_close(got[0], want[0], rtol=0, atol=0)
    torch.testing.assert_close(got[1], want[1], rtol=RTOL, atol=ATOL)
    return got


SIZES = [(1, 1), (3, 2), (2, 7), (5, 31), (4, 257), (7, 1000), (3, 4097), (2, 20481), (130, 3001), (2, 151936), (1, 248320), (3, 300001)]


@pytest.mark.parametrize("B,V", SIZES)
@pytest.mark.parametrize("settings", [(1.0,), (0.7, 0, 0.9), (1.3, 20), (0.9, 0, 1.0, 0.05), (0.8, 50, 0.95, 0.02), (0.0,), (1e-3,), (50.0, 0, 0.99)])
def test_draws_equal_the_expression(B, V, settings):
    same(*make(B, V, seed=B + V), *settings)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("spare", [0, 1, 3, 8])
def test_types_and_strides(dtype, spare):
    z, u = make(9, 4111, dtype, spare, spare)
    for s in ((1.0,), (0.8, 40, 0.9, 0.01)):
        same(z, u, *s)
    same(z[::2], u[::2], 0.8, 0, 0.9)
    wide, u = make(6, 500, dtype, 3)
    same(wide.t().contiguous().t(), u, 0.8, 30, 0.9)          # columns side by side: copied
    same(wide[:, 1:], u, 0.8, 30, 0.9)                        # rows that begin off the 16-byte boundaries


def test_settings_that_are_not_numbers_are_off_and_expanded_rows():
    z, u = make(6, 5003, seed=9)
    nan = float("nan")
    for s in ((1.0, 0, 1.0, nan), (1.0, 0, nan, 0.0), (0.8, 20, nan, nan), (0.8, 20, 0.9, torch.full((6,), nan, device="cuda"))):
        same(z, u, *s)
    a = sampling.sample(z, u, 0.8, 20)
    b = sampling.sample(z, u, 0.8, 20, nan, nan)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    same(z[:1].expand(6, 5003), u, 0.8, 0, 0.9)


@pytest.mark.parametrize("V,dtype", [(24601, torch.float32), (40003, torch.bfloat16), (151936, torch.float32)])
@pytest.mark.parametrize("top_p", [1e-6, 0.3, 0.9, 0.95, 0.9999])
def test_nuclei_of_long_rows_that_have_a_cta_each(V, dtype, top_p):
    """Rows of which a sample says roughly where the nucleus ends: usual ones, sharp and flat ones, and such that the sample misleads."""
    B = 80                                                     # more than half the SMs: no clusters
    z, u = make(B, V, dtype, seed=V)
    same(z, u, 0.7, 0, top_p)
    z = z.clone()
    z[0] = 1.0                                                 # all equal
    z[1, 1:] = -float("inf")
    z[2] = torch.where(torch.arange(V, device="cuda") % 2 == 0, 0.0, 3.0)
    z[3] *= 30
    z[4] *= 0.01
    z[5] = float("nan")
    z[6, ::3] = float("nan")
    z[7, V // 2:] = -float("inf")
    z[8] = torch.arange(V, device="cuda") / V                  # rising
    z[9, 17] = 1e30
    z[10, 17] = float("inf")
    z[11] = -1e30
    every = torch.arange(V, device="cuda") // (128 if dtype == torch.float32 else 256) % 8
    for i in range(8):                                         # one run of eight unlike the others: a sample of those sees another row
        z[12 + i] = torch.where(every == i, z[12 + i] - 6, z[12 + i])
        z[20 + i] = torch.where(every == i, z[20 + i] + 4, z[20 + i])
    z[28:40] = z[28:40].round()                                # many equal ones
    same(z, u, 0.7, 0, top_p)
    same(z, u, 1.3, 3000, top_p, 1e-4)
    same(z, u, torch.linspace(0.2, 3.0, B, device="cuda"), 0, top_p, 1e-3)


def test_settings_of_their_own_for_each_row():
    B, V = 48, 5003
    z, u = make(B, V, seed=5)
    g = torch.Generator().manual_seed(1)
    pick = lambda *v: torch.tensor(v)[torch.randint(len(v), (B,), generator=g)].cuda()        # noqa: E731
    T, k = pick(0.0, 0.5, 1.0, 2.0, float("nan")), pick(0, -1, 1, 3, 100, 5003, 9999)
    p, m = pick(1.0, 0.0, 0.1, 0.9, 0.999, 1.5, -1.0), pick(0.0, 0.01, 0.3, 1.0, 2.0)
    same(z, u, T, k, p, m)
    same(z, u, T, k.to(torch.int32), 1.0, m)
    same(z, u.double(), 1.0, k, p, 0.0)
    for u1 in (0.0, 1.0, 2.0, -1.0, float("nan"), 1 - 2.0 ** -24):
        same(z, torch.full_like(u, u1), 0.9, k, p, m)


@pytest.mark.parametrize("V", [600, 40000])
def test_equal_logits_stay_or_go_together(V):
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randint(-3, 4, (16, V), device="cuda", generator=g).float()        # thousands of each value
    u = torch.rand(16, device="cuda", generator=g)
    for s in ((1.0,), (1.0, 5), (1.0, 0, 0.5), (0.5, 0, 0.999), (1.0, V // 2, 0.3, 0.1), (0.0,)):
        same(z, u, *s)
    same(torch.zeros_like(z), u, 1.0, 3, 0.2)
    z[:, ::2] *= -1                                                               # zeros of both signs
    same(z, u, 0.7, 10, 0.8)


def test_nearby_logits_are_told_apart():
    """Thousands of different logits within an eighth of a nat: the class of a histogram does not hold the answer alone."""
    g = torch.Generator(device="cuda").manual_seed(3)
    z = 5 + 0.01 * torch.randn((8, 30000), device="cuda", generator=g)
    u = torch.rand(8, device="cuda", generator=g)
    for s in ((1.0, 300), (1.0, 0, 0.3), (1.0, 0, 0.9), (1.0, 20000, 0.5), (0.01, 7, 0.5, 0.2)):
        same(z, u, *s)


def test_masks_and_what_is_no_number():
    z, u = make(8, 3000, seed=4)
    inf, low = float("inf"), torch.finfo(torch.float32).min
    z[0] = -inf
    z[1, 100:] = -inf
    z[2, 7:] = low
    z[3] = low
    z[4, ::3] = float("nan")
    z[5, 11] = z[5, 1200] = inf
    z[6] = float("nan")
    z[7, :2999] = -inf
    for s in ((1.0,), (0.8, 50, 0.9, 0.05), (0.0,), (1.0, 200), (1.0, 0, 0.5)):
        tokens, lp = same(z, u, *s)
        assert int(tokens[0]) == 0 and float(lp[0]) == -inf and int(tokens[6]) == 0
        assert int(tokens[7]) == 2999 and int(tokens[1]) < 100


def test_frequencies_follow_the_distribution():
    """20000 draws from 6 tokens: a count is off its mean by 5 of its deviations (once in a million)."""
    p = torch.tensor([0.4, 0.3, 0.15, 0.1, 0.04, 0.01], device="cuda")
    n = 20000
    u = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    tokens, _ = sampling.sample(p.log().expand(n, 6), u)
    count = torch.bincount(tokens, minlength=6).float()
    assert bool(((count - n * p).abs() < 5 * (n * p * (1 - p)).sqrt()).all())


def test_rows_do_not_depend_on_the_batch_and_runs_repeat():
    z, u = make(64, 30011, seed=6)
    all_rows = sampling.sample(z, u, 0.9, 0, 0.95)
    for i in (0, 31, 63):
        one = sampling.sample(z[i:i + 1], u[i:i + 1], 0.9, 0, 0.95)
        assert int(one[0]) == int(all_rows[0][i])
    again = sampling.sample(z, u, 0.9, 0, 0.95)
    assert torch.equal(again[0], all_rows[0]) and torch.equal(again[1], all_rows[1])


def test_out_streams_and_captured_graphs():
    z, u = make(12, 9001, seed=7)
    out = (torch.full((12,), -1, device="cuda", dtype=torch.int32), torch.zeros(12, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sampling.sample(z, u, 0.8, 40, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert got[0] is out[0]
    same(z, u, 0.8, 40, out=out)
    graphs = []
    for s in ((0.8, 0, 0.9), (1.0, 30)):
        o = (torch.empty_like(out[0]), torch.empty_like(out[1]))
        sampling.sample(z, u, *s, out=o)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            sampling.sample(z, u, *s, out=o)
        graphs.append((g, s, o))
    z2, u2 = make(12, 9001, seed=8)
    z.copy_(z2)
    u.copy_(u2)
    for g, _, _ in graphs:
        g.replay()
    for _, s, o in graphs:
        torch.testing.assert_close(o[0], sampling.sample_ref(z, u, *s)[0], rtol=0, atol=0)


def test_drawn_numbers_of_the_device():
    """Without uniforms: a hash of seed, step and row; another step or seed gives other numbers, the same ones the same."""
    n, V = 4096, 64
    z = torch.zeros((n, V), device="cuda")
    step = torch.zeros(1, device="cuda", dtype=torch.int32)

    def once(seed):
        out = torch.empty(n, device="cuda", dtype=torch.int32), torch.empty(n, device="cuda")
        sampling.draw_raw(z, None, 1.0, 0, 1.0, 0.0, *out, seed=seed, step=step)
        return out[0]
    a, b = once(1), once(2)
    assert torch.equal(a, once(1)) and not torch.equal(a, b)
    step += 1
    c = once(1)
    assert not torch.equal(a, c)
    for x in (a, b, c):
        count = torch.bincount(x, minlength=V).float()
        assert bool(((count - n / V).abs() < 6 * (n / V) ** 0.5).all())
    assert float((a == c).float().mean()) < 0.05


@pytest.mark.parametrize("B,V", [(1, 151936), (5, 4001), (130, 32000)])
def test_noise_is_that_of_the_engines_other_draws(B, V):
    """Without restrictions the tokens of the rollout engine's kernel; with them, where that token stays, the same one."""
    import ctypes
    from arctic_platform_b200.engine.sampler import _fn
    from arctic_platform_b200.ops import _lib
    z, _ = make(B, V, seed=11)
    T = torch.full((B,), 0.8, device="cuda")
    step = torch.full((1,), 7, device="cuda", dtype=torch.int32)
    seed = torch.full((1,), 99, device="cuda", dtype=torch.int32)
    new = lambda: (torch.empty(B, device="cuda", dtype=torch.int32), torch.empty(B, device="cuda"))      # noqa: E731
    want, got, held = new(), new(), new()
    _lib.check(_fn("sample")(_lib.ptr(z), z.stride(0), _lib.ptr(T), B, V, ctypes.c_uint(99), _lib.ptr(step), _lib.ptr(want[0]), _lib.ptr(want[1]),
                             _lib.stream_ptr()), "sample")
    sampling.draw_raw(z, None, T, 0, 1.0, 0.0, *got, seed=seed, step=step)
    torch.testing.assert_close(got[0], want[0], rtol=0, atol=0)
    torch.testing.assert_close(got[1], want[1], rtol=RTOL, atol=2 * ATOL)
    sampling.draw_raw(z, None, T, 0, 1.0, 0.05, *held, seed=99, step=step)
    x = z.double() / 0.8
    stays = (x - x.amax(-1, keepdim=True)).gather(1, want[0].long()[:, None])[:, 0] >= torch.log(torch.tensor(0.05)).double()
    assert bool((held[0] == want[0])[stays].all()) and bool((held[0] != want[0])[~stays].all())
    kept = (x - x.amax(-1, keepdim=True)).gather(1, held[0].long()[:, None])[:, 0]
    assert bool((kept >= torch.log(torch.tensor(0.05)).double()).all())


def test_refusals():
    z, u = make(4, 50)
    for bad in ((z[0], u), (z.double(), u), (z, u[:3]), (z, u.half()), (z, u.cpu()), (z, u, torch.ones(3, device="cuda")),
                (z, u, 1.0, torch.ones(4, device="cuda")), (z, u, 1.0, 0, torch.ones(4, device="cuda", dtype=torch.int32)),
                (z, u, torch.ones(4)), (torch.zeros((1, sampling.MOST_VOCABULARY + 1), device="cuda"), u[:1])):
        with pytest.raises(ValueError):
            sampling.sample(*bad)
    with pytest.raises(ValueError):
        sampling.sample(z, u, out=(torch.empty(4, device="cuda"), torch.empty(4, device="cuda")))
    empty = sampling.sample(z[:0], u[:0], 0.8)
    assert empty[0].shape == (0,)
