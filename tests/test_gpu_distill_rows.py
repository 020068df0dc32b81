"""Hidden states that are copied before the kernels read them: dense ones off the 16-byte boundary, a single row of any stride."""
import pytest
import torch

from arctic_platform_b200.ops import distill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("off", [1, 2, 7, 8])
@pytest.mark.parametrize("N", [1, 6])
def test_hidden_states_off_their_boundary(N, off):
    V, H, K = 256, 64, 3
    g = torch.Generator(device="cuda").manual_seed(3)
    w = (torch.randn((V, H), device="cuda", generator=g) / 8).bfloat16()
    h = torch.randn((N, H), device="cuda", generator=g).bfloat16()
    ids = torch.randint(V, (N, K), device="cuda", generator=g)
    lq = torch.log_softmax(torch.randn((N, K + 1), device="cuda", generator=g), -1)

    def run(x):
        value = distill.lm_head_distill(x, w, ids[:, 0], ids, lq[:, :K], lq[:, K])[0]
        return value.detach(), torch.autograd.grad(value.sum(), x)[0]

    want = run(h.clone().requires_grad_(True))
    flat = torch.zeros(N * H + off, device="cuda", dtype=torch.bfloat16)
    flat[off:] = h.reshape(-1)
    wide = torch.zeros((N, H + 137), device="cuda", dtype=torch.bfloat16)
    wide[:, off:off + H] = h
    for x in (flat[off:].view(N, H), wide[:, off:off + H]):
        got = run(x.detach().requires_grad_(True))
        assert torch.equal(got[0], want[0])
        torch.testing.assert_close(got[1], want[1], rtol=2.0 ** -7, atol=1e-6)       # parts of the vocabulary add up in any order
