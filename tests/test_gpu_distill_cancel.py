"""Distillation through the lm head where the terms of a gradient cancel, against 64 bits."""
import pytest
import torch

from arctic_platform_b200.ops import distill

pytestmark = pytest.mark.gpu


def data(gap, N=40, V=800, H=64, K=5):
    """One named token ``gap`` nats above all others, by a column of its own."""
    g = torch.Generator(device="cuda").manual_seed(21)
    w = (torch.randn((V, H), device="cuda", generator=g) / 8).bfloat16()
    h = torch.randn((N, H), device="cuda", generator=g).bfloat16()
    ids = torch.stack([torch.randperm(V, device="cuda", generator=g)[:K] for _ in range(N)])
    ids[ids == 7] = 8
    ids[:, 2] = 7
    w[:, 0] = 0
    w[7, 0] = 1
    h[:, 0] = gap
    lq = torch.log_softmax(torch.randn((N, K + 1), device="cuda", generator=g), -1)
    return h, w, ids[:, 0].clone(), ids, lq[:, :K].contiguous(), lq[:, K].contiguous()


def gradients(h, w, labels, ids, lq, rest, reverse, up):
    z = (h.double() @ w.double().t()).requires_grad_(True)
    eye = torch.eye(w.shape[0], dtype=torch.float64, device="cuda")
    value = distill.distill_ref(z, eye, labels, ids, lq, rest, 1.0, reverse, False, torch.float64)[0]
    (d,) = torch.autograd.grad(value, z, up.double())
    return d, d @ w.double(), d.t() @ h.double()


@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("kept", [False, True])
def test_a_student_that_is_sure_has_no_reverse_gradient(kept, with_rest, monkeypatch):
    """All mass on one token: p (log p - log q + 1 - E) vanishes with the mass of the others, here e^-50.  A term is below 60 and 64-bit sums leave
    2^-50 of it, far below 1e-12."""
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: kept)
    h, w, labels, ids, lq, rest = data(50)
    rest = rest if with_rest else None
    up = torch.randn(40, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    d, dh, dw = gradients(h, w, labels, ids, lq, rest, 1.0, up)
    assert float(d.abs().max()) < 1e-16            # 800 e^-49 of mass, times 60, times an upstream gradient below 4
    hl, wl = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    value = distill.lm_head_distill(hl, wl, labels, ids, lq, rest, 1.0, 1.0)[0]
    got = torch.autograd.grad(value, (hl, wl), up)
    for a, b in zip(got, (dh, dw)):
        assert float((a.double() - b).abs().max()) < 1e-12


@pytest.mark.parametrize("kept", [False, True])
def test_the_log_prob_of_a_sure_token_has_no_gradient(kept, monkeypatch):
    """1 - p is the others' mass, e^-50 again, and not what a log-sum-exp of 50 loses in 32 bits."""
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: kept)
    h, w, _, ids, lq, rest = data(50)
    h[:20, 1:] /= 64
    # The label among the named tokens: 800 e^-49 of mass, times 50.  Not among them: its logit in the log-sum-exp is the product's, off by
    # H 2^-23 of its sum of magnitudes (60) at most, as is then 1 - p, times 50 again.
    for named, bound in ((ids, 1e-15), (torch.where(ids == 7, 9, ids), 64 * 2.0 ** -23 * 60 * 50)):
        hl, wl = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        lp = distill.lm_head_distill(hl, wl, torch.full((40,), 7, device="cuda"), named, lq, rest)[1]
        for a in torch.autograd.grad(lp.sum(), (hl, wl)):
            assert float(a.abs().max()) < bound


@pytest.mark.parametrize("reverse", [0.0, 0.5, 1.0])
def test_a_student_that_is_its_teacher(reverse):
    """All tokens named, the teacher's numbers the student's rounded to fp32, logits of whole numbers and so exact: the gradient is what that
    rounding makes, 1e-7 of p, and has the relative error of any other (d(logits) in bf16, sums of H products, results in bf16)."""
    g = torch.Generator(device="cuda").manual_seed(5)
    N, V, H = 24, 64, 64
    w = torch.randint(-1, 2, (V, H), device="cuda", generator=g).bfloat16()
    h = (torch.randint(-1, 2, (N, H), device="cuda", generator=g) / 2).bfloat16()
    lq = torch.log_softmax(h.double() @ w.double().t(), -1).float()
    ids = torch.arange(V, device="cuda").expand(N, V).contiguous()
    d, dh, dw = gradients(h, w, ids[:, 0], ids, lq, None, reverse, torch.ones(N, device="cuda"))
    assert 0 < float(d.abs().max()) < 1e-6
    hl, wl = h.requires_grad_(True), w.requires_grad_(True)
    value = distill.lm_head_distill(hl, wl, ids[:, 0], ids, lq, None, 1.0, reverse)[0]
    got = torch.autograd.grad(value.sum(), (hl, wl))
    # besides the roundings: 64-bit terms of size 1 leave 2^-50
    for a, b, s in zip(got, (dh, dw), (d.abs() @ w.double().abs(), d.abs().t() @ h.double().abs())):
        assert bool(((a.double() - b).abs() <= 1.1 * 2.0 ** -8 * s + 2.0 ** -8 * b.abs() + 1e-13).all())
