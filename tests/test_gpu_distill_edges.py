"""Distillation through the lm head at the edges of its range, against 64 bits.  Tolerances as in the other tests of it: a logit of the tokens not named
is off by ERR at most (H 2^-23 of its sum of magnitudes, below 30 here), d(logits) is rounded to bf16 and so is a gradient."""
import pytest
import torch

from arctic_platform_b200.ops import distill

pytestmark = pytest.mark.gpu
ERR = 1e-3


def gradients(h, w, labels, ids, lq, rest, reverse, ups):
    """Values, gradients of hidden and weight, and their sums of magnitudes, in 64 bits."""
    z = (h.double() @ w.double().t()).requires_grad_(True)
    eye = torch.eye(w.shape[0], dtype=torch.float64, device="cuda")
    out = distill.distill_ref(z, eye, labels, ids, lq, rest, 1.0, reverse, True, torch.float64)
    (d,) = torch.autograd.grad([o for o, u in zip(out, ups) if u is not None], z, [u.double() for u in ups if u is not None])
    return out, d, d @ w.double(), d.t() @ h.double(), d.abs() @ w.double().abs(), d.abs().t() @ h.double().abs()


def sure_student(gap, N=40, V=800, H=64, K=5):
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
    labels = torch.randint(V, (N,), device="cuda", generator=g)
    labels[::4] = 7
    return h, w, labels, ids, lq[:, :K].contiguous(), lq[:, K].contiguous()


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("reverse", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("gap", [50, 68, 80, 92, 104, 300])
def test_others_far_below_a_named_token(gap, reverse, kept, monkeypatch):
    """Their probabilities leave the range of fp32, their part of the gradient does not: (1 - reverse) times the mass that the teacher gives them."""
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: kept)
    h, w, labels, ids, lq, rest = sure_student(gap)
    N = len(h)
    g = torch.Generator(device="cuda").manual_seed(1)
    for which in ((1, 0, 0), (1, 1, 0), (1, 1, 1)):
        ups = [torch.randn(N, device="cuda", generator=g) if x else None for x in which]
        want, d, dh, dw, sh, sw = gradients(h, w, labels, ids, lq, rest, reverse, ups)
        hl, wl = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        got = distill.lm_head_distill(hl, wl, labels, ids, lq, rest, 1.0, reverse)
        for a, b in zip(got, want):
            torch.testing.assert_close(a.double(), b, rtol=2.0 ** -20, atol=4 * ERR)
        grads = torch.autograd.grad([o for o, u in zip(got, ups) if u is not None], (hl, wl), [u for u in ups if u is not None])
        for a, b, s in zip(grads, (dh, dw), (sh, sw)):
            off = (a.double() - b).abs()
            bound = (2 * 2.0 ** -8 + 4 * ERR) * s + 2.0 ** -8 * b.abs() + 1e-12
            assert bool((off <= bound).all()), float((off / s.clamp_min(1e-9)).max())
    if reverse < 1:                            # what the others get is there to be lost
        others = d.clone()
        others.scatter_(1, ids, 0.0)
        assert float(others.abs().sum(-1).min()) > 1e-3 * (1 - reverse)
