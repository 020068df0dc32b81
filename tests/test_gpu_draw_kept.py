"""Draws by the engines' noise under every restriction: the token is that of an unrestricted draw from the row in which what the restrictions leave
out (by the expression in 64 bits) is masked, to the bit, as a token's noise does not depend on the others.  A log-probability is that of the
whole row: 64-bit sums, rounded once to fp32 (2^-24 of it), against the expression's."""
import pytest
import torch

from arctic_platform_b200.ops import sampling

pytestmark = pytest.mark.gpu


def kept(z, T, k, p, m):
    """Tokens that stay, ``[B, V]``: the definition in 64 bits."""
    z = z.double()
    z = torch.where(torch.isnan(z), -float("inf"), z)
    B, V = z.shape
    column = lambda x: torch.as_tensor(x, dtype=torch.float32, device=z.device).double().expand(B)[:, None]       # noqa: E731
    T, p, m = column(T), column(p), column(m)
    k = torch.as_tensor(k, device=z.device).long().expand(B)[:, None]
    T = torch.where(T > 0, T, 1.0)
    most = z.amax(-1, keepdim=True)
    x = torch.where(z == most, 0.0, (z - most) / T)
    order = torch.sort(z, dim=-1, descending=True).values
    keep = z >= order.gather(1, torch.where((k > 0) & (k < V), k, V) - 1)
    keep &= (m <= 0) | (x >= torch.log(m.clamp_max(1.0)))
    value, rank = torch.sort(z, dim=-1, descending=True, stable=True)
    run = torch.where(keep, x.exp(), 0.0).gather(1, rank).cumsum(-1)
    first = torch.searchsorted(-value.contiguous(), -value.contiguous())
    larger = torch.where(first > 0, run.gather(1, (first - 1).clamp_min(0)), 0.0)
    stays = (larger < p * run[:, -1:]) | (p >= 1) | (value == most)
    return keep & torch.zeros_like(keep).scatter(1, rank, stays)


def draw(z, T, k, p, m, seed, step):
    B = z.shape[0]
    out = torch.empty(B, device="cuda", dtype=torch.int32), torch.empty(B, device="cuda")
    row = lambda x, dtype: torch.as_tensor(x, dtype=dtype, device="cuda").expand(B).contiguous()                     # noqa: E731
    at = torch.full((1,), step, device="cuda", dtype=torch.int32)
    sampling.draw_raw(z, None, row(T, torch.float32), row(k, torch.int32), row(p, torch.float32), row(m, torch.float32), *out, seed=seed, step=at)
    return out


def make(B, V, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = 2 * torch.randn((B, V), device="cuda", generator=g)
    ids = torch.randint(V, (B, min(40, V)), device="cuda", generator=g)
    return z.scatter_reduce_(1, ids, 4 + 8 * torch.rand(ids.shape, device="cuda", generator=g), "amax").to(dtype)


SETTINGS = [(1.0, 0, 0.9, 0.0), (0.7, 50, 1.0, 0.0), (1.3, 0, 0.99, 0.0), (1.0, 400, 0.95, 0.001), (0.6, 0, 1.0, 0.1), (1.0, 20, 0.5, 0.05),
            (2.0, 0, 0.5, 0.0), (0.0, 20, 0.5, 0.05)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,V", [(1, 5), (2, 777), (5, 30011), (3, 151936), (100, 24600), (80, 40003)])
def test_restricted_draws_by_noise(B, V, dtype):
    z = make(B, V, dtype, B + V)
    for i, (T, k, p, m) in enumerate(SETTINGS):
        mask = kept(z, T, k, p, m)
        got = draw(z, T, k, p, m, 1234 + i, 3 * i)
        want = draw(z.masked_fill(~mask, -float("inf")), T, 0, 1.0, 0.0, 1234 + i, 3 * i)
        assert torch.equal(got[0], want[0])
        x = z.double() / (T if T > 0 else 1.0)
        lp = torch.log_softmax(x, -1).gather(1, got[0].long()[:, None])[:, 0]
        torch.testing.assert_close(got[1].double(), lp, rtol=2.0 ** -22, atol=1e-9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_with_settings_of_their_own(dtype):
    B, V = 90, 32003
    z = make(B, V, dtype, 7)
    g = torch.Generator().manual_seed(1)
    pick = lambda *v: torch.tensor(v)[torch.randint(len(v), (B,), generator=g)].cuda()        # noqa: E731
    T, k, p, m = pick(0.0, 0.5, 1.0, 2.0), pick(0, 1, 3, 100, 40000), pick(1.0, 0.1, 0.9, 0.999), pick(0.0, 0.01, 0.3)
    got = draw(z, T, k, p, m, 5, 6)
    # restrictions of a greedy row are off
    want = draw(z.masked_fill(~kept(z, T, k, p, m), -float("inf")), T, 0, 1.0, 0.0, 5, 6)
    assert torch.equal(got[0], want[0])
    assert torch.equal(got[0][T == 0].long(), z.float().argmax(-1)[T == 0])


@pytest.mark.parametrize("T,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 0, 0.95, 0.0), (1.0, 50, 1.0, 0.0), (1.0, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0)])
@pytest.mark.parametrize("B,V", [(3, 1000), (2, 151936), (140, 32000)])
def test_log_probabilities_to_the_rounding_of_fp32(B, V, T, k, p, m):
    """With given numbers too: masses and sums of 64 bits (a mass is off by 4e-11), so that only the result's rounding is left."""
    z = make(B, V, torch.float32, 3)
    u = torch.rand(B, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    tokens, lp = sampling.sample(z, u, T, k, p, m)
    t = float(torch.tensor(T, dtype=torch.float32)) or 1.0
    want = torch.log_softmax(z.double() / t, -1).gather(1, tokens.long()[:, None])[:, 0]
    torch.testing.assert_close(lp.double(), want, rtol=2.0 ** -24, atol=1e-9)
