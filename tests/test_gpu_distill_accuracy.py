"""How exact distillation through the lm head is, against 64 bits.

Values.  The logits of the named tokens are 64-bit sums of eight products each (fp32: 8 2^-24 of their magnitudes, below 4: 2e-6 at most and either
way).  Those of the others are running sums of H / 16 steps, each off by 2^-24 of a partial sum (below 16: 2^-20), which for H = 1024 and
independent errors makes 2^-17 of a logit; a log-probability has the log-sum-exp's error beside its own: 2^-16 = 1.5e-5 in all, which a divergence
takes over per unit of mass.  Bound: 2e-5 of 1 + the value.

Gradients of a real vocabulary.  d(logits) is rounded to bf16 (others that are kept twice) and so is the result: each by 2^-8 at most, 2^-8 / sqrt(3)
in the mean of a worst mantissa, independently: 2^-8 sqrt(3 / 3) = 2^-8 of the norm for three of them."""
import pytest
import torch

from arctic_platform_b200.ops import distill

pytestmark = pytest.mark.gpu


def make(N, V, H, K, seed=0):
    """Rows in which a few tokens stand out; a teacher near the student."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((V, H), device="cuda", generator=g) * (1.2 / H ** 0.5)).bfloat16()
    ids = torch.randint(V, (N, 4), device="cuda", generator=g)
    h = torch.randn((N, H), device="cuda", generator=g) + sum(s * w[ids[:, i]].float() for i, s in enumerate((6, 5, 4, 3)))
    h = h.bfloat16()
    z = h.double() @ w.double().t()
    t = torch.log_softmax(z + torch.randn(z.shape, device="cuda", generator=g), -1)
    lq, top = t.topk(K, -1)
    rest = torch.logsumexp(t.scatter(1, top, -float("inf")), -1)
    labels = torch.where(torch.arange(N, device="cuda") % 2 == 0, ids[:, 0], torch.randint(V, (N,), device="cuda", generator=g))
    return h, w, labels, top.to(torch.int32), lq.float(), rest.float(), z


@pytest.mark.parametrize("reverse", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("N,V,H,K", [(37, 32000, 256, 8), (5, 8192, 1024, 64), (130, 4096, 512, 20)])
def test_values(N, V, H, K, with_rest, reverse):
    h, w, labels, ids, lq, rest, z = make(N, V, H, K, N)
    rest = rest if with_rest else None
    got = distill.lm_head_distill(h, w, labels, ids, lq, rest, 1.0, reverse)
    log_p = torch.log_softmax(z, -1)
    named = log_p.gather(1, ids.long())
    P = [named] + ([torch.logsumexp(log_p.scatter(1, ids.long(), -float("inf")), -1, keepdim=True)] if with_rest else [])
    Q = [lq.double()] + ([rest.double()[:, None]] if with_rest else [])
    P, Q = torch.cat(P, -1), torch.cat(Q, -1)
    value = (1 - reverse) * (Q.exp() * (Q - P)).sum(-1) + reverse * (P.exp() * (P - Q)).sum(-1)
    entropy = -(log_p.exp() * log_p).sum(-1)
    for a, b in zip(got, (value, log_p.gather(1, labels.long()[:, None])[:, 0], entropy)):
        off = (a.double() - b).abs()
        assert bool((off <= 2e-5 * (1 + b.abs())).all()), float(off.max())


@pytest.mark.parametrize("N,V,H,K,kept", [(549, 151936, 1024, 20, True), (549, 151936, 1024, 20, False), (300, 151936, 2560, 64, True), (37, 32000, 256, 8, False)])
@pytest.mark.parametrize("with_rest,reverse", [(True, 0.5), (False, 0.0)])
def test_gradients_of_a_real_vocabulary(N, V, H, K, kept, with_rest, reverse, monkeypatch):
    """More than a thousand records a row, several waves of tiles, d_hidden in parts of the vocabulary."""
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: kept)
    h, w, labels, ids, lq, rest, z = make(N, V, H, K, N)
    rest = rest if with_rest else None
    g = torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) / N
    hl, wl = h.requires_grad_(True), w.requires_grad_(True)
    value = distill.lm_head_distill(hl, wl, labels, ids, lq, rest, 1.0, reverse, False)[0]
    dh, dw = torch.autograd.grad(value, (hl, wl), g)
    # d value / d log P of every class, then of its tokens: log P is the log-sum-exp of the class
    lp = torch.log_softmax(z, -1)
    del z
    at = ids.long()
    named, lq = lp.gather(1, at), lq.double()
    by = -(1 - reverse) * lq.exp() + reverse * named.exp() * (1 + named - lq)
    total = by.sum(-1, keepdim=True)
    d = torch.zeros_like(lp)
    if with_rest:
        left = torch.logsumexp(lp.scatter(1, at, -float("inf")), -1, keepdim=True)
        r = rest.double()[:, None]
        of_rest = -(1 - reverse) * r.exp() + reverse * left.exp() * (1 + left - r)
        total = total + of_rest
        d += (lp - left).exp() * of_rest
    d.scatter_(1, at, by)
    d -= lp.exp() * total
    d *= g.double()[:, None]
    for a, b in ((dh, d @ w.detach().double()), (dw, d.t() @ h.detach().double())):
        assert float((a.double() - b).norm() / b.norm()) < 2.0 ** -8
    # a row's roundings do not average over others
    rows, want = (dh.double() - d @ w.detach().double()).norm(dim=-1), (d.abs() @ w.detach().double().abs()).norm(dim=-1)
    assert bool((rows <= 3 * 2.0 ** -8 * want).all())
