"""What a backward pass keeps and forms at a time where the caller bounds its memory or wants the same bits each time."""
import pytest
import torch

from arctic_platform_b200.ops import distill
from arctic_platform_b200.utils import memory_budget

pytestmark = pytest.mark.gpu


def data(N, V=1024, H=64, K=4):
    g = torch.Generator(device="cuda").manual_seed(2)
    h = torch.randn((N, H), device="cuda", generator=g).bfloat16().requires_grad_(True)
    w = (torch.randn((V, H), device="cuda", generator=g) / 8).bfloat16().requires_grad_(True)
    ids = torch.randint(V, (N, K), device="cuda", generator=g)
    lq = torch.log_softmax(torch.randn((N, K + 1), device="cuda", generator=g), -1)
    return h, w, ids[:, 0], ids, lq[:, :K].contiguous(), lq[:, K].contiguous()


def kept(value, N, V):
    return [t for t in value.grad_fn.saved_tensors if t is not None and tuple(t.shape) == (N, V)]


@pytest.fixture
def deterministic():
    torch.use_deterministic_algorithms(True, warn_only=True)
    yield
    torch.use_deterministic_algorithms(False)


def test_a_caller_that_bounds_memory_keeps_no_exponentials(monkeypatch):
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: True)
    args = data(300)
    assert len(kept(distill.lm_head_distill(*args)[0], 300, 1024)) == 1
    assert not kept(distill.lm_head_distill(*args, bwd_chunk=128)[0], 300, 1024)


def test_deterministic_algorithms_do_not_ask_for_spare_memory(deterministic, monkeypatch):
    """The rows at a time are those of a device without any to spare."""
    chunks, rows = [], distill._bwd_rows
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: True)
    monkeypatch.setattr(memory_budget, "spare_bytes", lambda device, wanted: wanted)
    monkeypatch.setattr(distill, "_bwd_rows", lambda *a: chunks.append(rows(*a)) or chunks[-1])
    args = data(9000)
    value = distill.lm_head_distill(*args, reverse=0.5)[0]
    assert not kept(value, 9000, 1024)
    torch.autograd.grad(value.sum(), args[:2])
    assert chunks == [rows(9000, 1024, 0)] and chunks[0] < 9000
