"""Draws with numbers at and next to 0: the first token that has any mass, however little, as the expression in 64 bits has it."""
import pytest
import torch

from arctic_platform_b200.ops import sampling

pytestmark = pytest.mark.gpu


def rows(B, V, low, seed=0):
    """Ordinary rows whose first third lies `low` nats below the rest, and whose very first tokens have no mass at all."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = 2 * torch.randn((B, V), device="cuda", generator=g)
    z[:, :V // 3] -= low
    z[:, :V // 50] = -float("inf")
    z[::2, :V // 40] = torch.finfo(torch.float32).min
    z[1::4, V // 50 + 1] = float("nan")
    return z


@pytest.mark.parametrize("B,V", [(1, 7), (3, 300), (2, 20481), (130, 4001), (2, 151936), (80, 40003)])
@pytest.mark.parametrize("low", [0, 45, 60, 90, 300, 600, 2000])
@pytest.mark.parametrize("settings", [(1.0,), (0.5,), (1.0, 0, 1.0, 1e-30), (1.3, 0, 1.0 - 2.0 ** -24), (1.0, 1 << 20)])
def test_numbers_next_to_0(B, V, low, settings):
    z = rows(B, V, low, seed=V + low)
    k = (min(settings[1], V - 1),) if len(settings) == 2 else settings[1:2]
    settings = settings[:1] + k + settings[2:]
    for u in (0.0, 1e-300, 1e-45, 1e-30, 2.0 ** -70, 2.0 ** -59, 2.0 ** -24):
        u = torch.full((B,), u, device="cuda", dtype=torch.float64)
        got, want = sampling.sample(z, u, *settings), sampling.sample_ref(z, u, *settings)
        assert torch.equal(got[0], want[0]), (got[0] - want[0]).nonzero()[:, 0].tolist()
        torch.testing.assert_close(got[1], want[1], rtol=2.0 ** -22, atol=1e-6)
    zero = torch.zeros(B, device="cuda")
    assert torch.equal(sampling.sample(z, zero, *settings)[0], sampling.sample_ref(z, zero, *settings)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_with_one_token_of_mass_and_shifted_rows(dtype):
    V = 30000
    z = torch.full((6, V), -float("inf"), device="cuda")
    z[0, 17], z[0, 29000] = -650.0, 0.0
    z[1, 17], z[1, 29000] = -1000.0, 0.0                      # less than e^-693 of the largest
    z[2] = 500.0                                              # sums of the first walk that are far from 1
    z[2, :100] = 400.0
    z[3] = -500.0
    z[3, :100] = -590.0
    z[4] = 3000.0                                             # and such that are not used
    z[4, :100] = 2910.0
    z[5, 5] = z[5, 28000] = float("inf")
    z = z.to(dtype)
    u = torch.zeros(6, device="cuda")
    got, want = sampling.sample(z, u), sampling.sample_ref(z, u)
    assert torch.equal(got[0], want[0]) and got[0].tolist() == [17, 29000, 0, 0, 0, 5]
