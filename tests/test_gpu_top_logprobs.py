"""The most likely tokens of rows of logits on a GPU against the expression in 64 bits: indices are equal; log-probabilities and the others' mass
come from fp32 sums of at most 300 elements a thread, 32 threads, 32 warps and 8 parts (each addition off by 2^-24: 2e-5 at most) of
approximate exponentials (3e-6)."""
import pytest
import torch

from arctic_platform_b200.ops import logprob

pytestmark = pytest.mark.gpu
ATOL, RTOL = 3e-5, 2.0 ** -22


def same(z, k, it=1.0):
    got = logprob.top_logprobs(z, k, it)
    want = logprob.top_logprobs_ref(z, k, it, torch.float64)
    torch.testing.assert_close(got[1], want[1], rtol=0, atol=0)
    torch.testing.assert_close(got[0], want[0], rtol=RTOL, atol=ATOL)
    # the others' share: its logarithm is near 0 where nothing is named, off by the sums' relative errors
    torch.testing.assert_close(got[2], want[2], rtol=RTOL, atol=ATOL)
    return got


def make(N, V, dtype=torch.float32, seed=0, spare=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = 2 * torch.randn((N, V + spare), device="cuda", generator=g)
    z[:, ::37] += 4 * torch.rand((N, len(range(0, V + spare, 37))), device="cuda", generator=g)
    return z.to(dtype)[:, :V]


@pytest.mark.parametrize("N,V", [(1, 1), (2, 5), (3, 64), (1, 1024), (5, 2049), (300, 1000), (1, 8193), (3, 32000), (40, 50001), (1, 151936), (2, 248320)])
@pytest.mark.parametrize("k", [1, 2, 20, 63, 256, 1024])
def test_top_equals_the_expression(N, V, k):
    same(make(N, V, seed=N + V), min(k, V))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("spare", [0, 1, 7])
def test_types_strides_and_ties(dtype, spare):
    z = make(20, 9003, dtype, spare, spare)
    for k in (1, 30, 500):
        same(z, k)
    same(z[::3], 12)
    same(z[:, 3:], 12)
    same(z.t().contiguous().t(), 12)
    same(torch.zeros_like(z), 40)                             # all equal: the first ones
    g = torch.Generator(device="cuda").manual_seed(3)
    few = torch.randint(-2, 3, (6, 20000), device="cuda", generator=g).to(dtype)
    few[:, ::2] *= -1
    for k in (5, 700, 1024):
        same(few, k)


@pytest.mark.parametrize("V", [3000, 60000])
def test_rising_and_falling_rows(V):
    """A row that rises fills the buffer again and again."""
    z = torch.arange(V, device="cuda").float()[None] / V
    for x in (z, z.flip(1), torch.cat([z, z.flip(1)])):
        for k in (1, 100, 1024):
            same(x * 20, k)


def test_temperatures():
    z = make(7, 5000)
    same(z, 25, 0.5)
    same(z, 25, torch.linspace(0.2, 3, 7, device="cuda"))
    same(z * 30, 25, 4.0)                                     # nearly all of the mass named
    same(z * 1e-3, 3)                                         # nearly none


def test_masks_and_what_is_no_number():
    inf = float("inf")
    z = make(7, 3001, seed=2)
    z[0] = -inf
    z[1, 5:] = -inf
    z[2, 3:] = torch.finfo(torch.float32).min
    z[3, ::2] = float("nan")
    z[4, 10] = z[4, 2000] = inf
    z[5] = torch.finfo(torch.float32).min
    z[6] = float("nan")
    got = logprob.top_logprobs(z, 8)
    want = logprob.top_logprobs_ref(z, 8, 1.0, torch.float64)
    for g, w in zip(got, want):
        keep = [1, 2, 3, 5]
        torch.testing.assert_close(g[keep], w[keep], rtol=RTOL, atol=ATOL)
    for r in (0, 6):
        assert bool((got[0][r] == -inf).all()) and float(got[2][r]) == -inf and got[1][r].tolist() == list(range(8))
    assert got[1][4, :2].tolist() == [10, 2000] and torch.allclose(got[0][4, :2], torch.tensor(0.5, device="cuda").log())
    assert bool((got[0][4, 2:] == -inf).all()) and float(got[2][4]) == -inf
    same(z[1:2], 1000)                                        # -inf among the named
    assert float(logprob.top_logprobs(make(1, 50), 50)[2]) == -inf


def test_streams_graphs_and_refusals():
    z = make(6, 4000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = logprob.top_logprobs(z, 9)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[1], logprob.top_logprobs_ref(z, 9)[1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = logprob.top_logprobs(z, 9)
    z.copy_(make(6, 4000, seed=5))
    g.replay()
    assert torch.equal(got[1], logprob.top_logprobs_ref(z, 9)[1])
    for bad in ((z[0], 3), (z, 0), (z, 4001), (z, 1025), (z.double(), 3), (z, 3, 0.0), (z, 3, -1.0), (z, 3, torch.ones(5, device="cuda"))):
        with pytest.raises(ValueError):
            logprob.top_logprobs(*bad)
    assert logprob.top_logprobs(z[:0], 3)[0].shape == (0, 3)
