"""A pass without gradients does none of a backward pass's work."""
import pytest
import torch

from arctic_platform_b200.ops import distill

pytestmark = pytest.mark.gpu


def test_values_without_gradients_keep_no_exponentials(monkeypatch):
    asked = []
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: asked.append(a) or True)
    g = torch.Generator(device="cuda").manual_seed(2)
    N, V, H, K = 512, 131072, 64, 4
    h = torch.randn((N, H), device="cuda", generator=g).bfloat16()
    w = (torch.randn((V, H), device="cuda", generator=g) / 8).bfloat16().requires_grad_(True)
    ids = torch.randint(V, (N, K), device="cuda", generator=g)
    lq = torch.log_softmax(torch.randn((N, K + 1), device="cuda", generator=g), -1)
    call = lambda x, y: distill.lm_head_distill(x, y, ids[:, 0], ids, lq[:, :K], lq[:, K])[0]          # noqa: E731
    with_grad = call(h, w)
    assert len(asked) == 1
    for off in (torch.no_grad, torch.inference_mode):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        with off():
            value = call(h.clone(), w)
        assert len(asked) == 1 and not value.requires_grad and torch.equal(value, with_grad.detach())
        assert torch.cuda.max_memory_allocated() - before < N * V                   # [N, V] in bf16 is twice that
    call(h, w.detach())
    assert len(asked) == 1
