"""The operators around the output distribution on CPU tensors: the expressions that the GPU tests compare with, against definitions written
out row by row, against differences, and their refusals."""
import math

import pytest
import torch

from arctic_platform_b200.engine.reference_sampler import LogitsProcessor, filter_logits
from arctic_platform_b200.ops import distill, logprob, sampling


def walk(z, u, T, k, p, m):
    """One row's draw, written out: sort, drop, walk."""
    V = len(z)
    if not T > 0:
        return max(range(V), key=lambda i: (z[i], -i))
    top = max(z)
    kth = sorted(z, reverse=True)[k - 1] if 0 < k < V else -math.inf
    keep = [i for i in range(V) if z[i] >= kth and (m <= 0 or (z[i] - top) / T >= math.log(min(m, 1.0)))]
    mass = {i: math.exp((z[i] - top) / T) for i in keep}
    if p < 1:
        total = sum(mass.values())
        mass = {i: w for i, w in mass.items() if sum(x for j, x in mass.items() if z[j] > z[i]) < p * total or z[i] == top}
    goal, run = u * sum(mass.values()), 0.0
    for i in sorted(mass):
        run += mass[i]
        if run > goal:
            return i
    return max(i for i in mass if mass[i] > 0)


@pytest.mark.parametrize("settings", [(1.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.2, 0, 0.8, 0.0), (0.9, 0, 1.0, 0.1), (1.5, 12, 0.6, 0.05),
                                      (0.0, 3, 0.5, 0.2), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 5.0)])
def test_draws_by_definition(settings):
    g = torch.Generator().manual_seed(1)
    z = torch.cat([2 * torch.randn((30, 40), generator=g), torch.randint(-2, 3, (30, 40), generator=g).float()])
    u = torch.rand(60, generator=g)
    tokens, lp = sampling.sample(z, u, *settings)
    T, k, p, m = (float(torch.tensor(x, dtype=torch.float32)) for x in settings)
    for i in range(60):
        assert int(tokens[i]) == walk(z[i].double().tolist(), float(u[i]), T, int(k), p, m)
    want = torch.log_softmax(z.double() / (T if T > 0 else 1.0), -1).gather(1, tokens.long()[:, None])[:, 0]
    torch.testing.assert_close(lp.double(), want, rtol=1e-6, atol=1e-6)


def test_what_stays_is_what_the_tensor_op_sampler_keeps():
    """Restrictions in the order of the tensor-op sampler; without equal logits both keep the same tokens."""
    g = torch.Generator().manual_seed(2)
    z = 2 * torch.randn((50, 60), generator=g)
    for T, k, p, m in ((0.8, 10, 0.9, 0.0), (1.0, 0, 0.7, 0.05), (1.3, 20, 1.0, 0.02)):
        for i in range(50):
            shaped = filter_logits(LogitsProcessor({"min_p": m}).after_temperature(z[i] / T), k, p)
            kept = set(torch.isfinite(shaped).nonzero()[:, 0].tolist())
            n = 400
            drawn = sampling.sample(z[i].expand(n, -1), (torch.arange(n) + 0.5) / n, T, k, p, m)[0]
            assert set(drawn.tolist()) <= kept
            heavy = torch.softmax(shaped, -1) > 2.0 / n
            assert set(heavy.nonzero()[:, 0].tolist()) <= set(drawn.tolist())


def test_masked_rows_out_and_refusals():
    inf = math.inf
    z = torch.tensor([[-inf, -inf, -inf], [math.nan, 1.0, -inf], [math.nan] * 3, [inf, 0.0, inf]])
    out = torch.empty(4, dtype=torch.int32), torch.empty(4)
    tokens, lp = sampling.sample(z, torch.tensor([0.3, 0.9, 0.1, 0.7]), 0.5, 2, 0.9, 0.1, out=out)
    assert tokens is out[0] and tokens.tolist() == [0, 1, 0, 2] and lp[0] == lp[2] == -inf and lp[1] == 0 and abs(float(lp[3]) + math.log(2)) < 1e-6
    u = torch.rand(4)
    for bad in ((z[0], u), (z.double(), u), (z, u[:3]), (z, u.half()), (z, u, torch.ones(3)), (z, u, 1.0, torch.ones(4)),
                (z, u, 1.0, 0, torch.ones(4, dtype=torch.int32)), (z[:, :0], u)):
        with pytest.raises(ValueError):
            sampling.sample(*bad)
    with pytest.raises(ValueError):
        sampling.sample(z, u, out=(torch.empty(4, dtype=torch.int32), torch.empty(3)))
    assert sampling.sample(z[:0], u[:0])[0].shape == (0,)


def test_top_logprobs_by_definition():
    g = torch.Generator().manual_seed(3)
    for z in (torch.randn((7, 50), generator=g), torch.randint(-2, 3, (7, 50), generator=g).float(), torch.randn((7, 50), generator=g).bfloat16()):
        for k, it in ((1, 1.0), (13, 0.7), (50, 2.0)):
            lp, ids, rest = logprob.top_logprobs(z, k, it)
            full = torch.log_softmax(z.double() * it, -1)
            for r in range(7):
                order = sorted(range(50), key=lambda i: (-float(z[r, i]), i))[:k]
                assert ids[r].tolist() == order
                torch.testing.assert_close(lp[r].double(), full[r, order], rtol=1e-6, atol=2e-6)
                others = full[r].clone()
                others[order] = -math.inf
                want = torch.logsumexp(others, 0)
                assert float(rest[r]) == pytest.approx(float(want), abs=2e-6) or (k == 50 and float(rest[r]) == -math.inf)
    for bad in ((z[0], 3), (z, 0), (z, 51), (z.long(), 3), (z, 3, 0.0), (z, 3, torch.ones(6))):
        with pytest.raises(ValueError):
            logprob.top_logprobs(*bad)


def case(dtype=torch.float64):
    g = torch.Generator().manual_seed(4)
    h, w = torch.randn((6, 16), generator=g).to(dtype), torch.randn((24, 16), generator=g).to(dtype)
    ids = torch.tensor([[1, 2, 3], [4, 4, 5], [-1, -1, -1], [7, 30, -1], [0, 1, 23], [9, 8, 9]])
    lq = torch.log_softmax(torch.randn((6, 4), generator=g).to(dtype), -1)
    return h, w, torch.arange(6), ids, lq[:, :3], lq[:, 3]


@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("reverse", [0.0, 0.3, 1.0])
def test_divergence_by_definition_and_by_differences(with_rest, reverse):
    h, w, labels, ids, lq, rest = case()
    f = lambda a, b: distill.distill_ref(a, b, labels, ids, lq, rest if with_rest else None, 1.3, reverse, True, torch.float64)   # noqa: E731
    value, lp, ent = f(h, w)
    logs = torch.log_softmax(h @ w.t() * 1.3, -1)
    for r in range(6):
        seen, F, R, left = set(), 0.0, 0.0, 1.0
        for k in range(3):
            v = int(ids[r, k])
            if not 0 <= v < 24 or v in seen:
                continue
            seen.add(v)
            p, q = float(logs[r, v]), float(lq[r, k])
            F += math.exp(q) * (q - p)
            R += math.exp(p) * (p - q)
            left -= math.exp(p)
        if with_rest:
            p, q = math.log(left), float(rest[r])
            F += math.exp(q) * (q - p)
            R += math.exp(p) * (p - q)
        assert float(value[r]) == pytest.approx((1 - reverse) * F + reverse * R, abs=1e-9)
        assert float(lp[r]) == pytest.approx(float(logs[r, r]))
        assert float(ent[r]) == pytest.approx(-float((logs[r].exp() * logs[r]).sum()))
    assert torch.autograd.gradcheck(f, (h.requires_grad_(True), w.requires_grad_(True)))


def test_lm_head_distill_on_cpu_and_refusals():
    h, w, labels, ids, lq, rest = case(torch.float32)
    value, lp, ent = distill.lm_head_distill(h.requires_grad_(True), w, labels, ids, lq, rest, torch.full((6,), 1.3), 0.3)
    want = distill.distill_ref(h.double(), w.double(), labels, ids, lq, rest, 1.3, 0.3, True, torch.float64)
    for a, b in zip((value, lp, ent), want):
        torch.testing.assert_close(a.double(), b, rtol=1e-4, atol=1e-5)
    assert float(value[2].detach()) != 0 and distill.lm_head_distill(h, w, labels, ids, lq)[0][2] == 0
    assert distill.lm_head_distill(h, w, labels, ids, lq, with_entropy=False)[2] is None
    f = distill.lm_head_distill
    for bad in (lambda: f(h[0], w, labels, ids, lq), lambda: f(h, w[:, :8], labels, ids, lq), lambda: f(h, w, labels[:3], ids, lq),
                lambda: f(h, w, labels, ids, lq[:, :2]), lambda: f(h, w, labels, ids.float(), lq), lambda: f(h, w, labels, ids, ids),
                lambda: f(h, w, labels, ids, lq, rest[:2]), lambda: f(h, w, labels, ids, lq, rest, torch.ones(5)),
                lambda: f(h, w, labels, ids, lq, rest, 1.0, -0.5), lambda: f(h, w, labels, ids, lq, rest, 1.0, 2.0)):
        with pytest.raises(ValueError):
            bad()


def test_a_class_without_mass_keeps_gradients_finite():
    h, w, labels, ids, lq, rest = case()
    lq = lq.clone()
    lq[0, 1], rest = -math.inf, rest.clone()
    rest[1] = -math.inf
    a = h.requires_grad_(True)
    value = distill.lm_head_distill(a, w, labels, ids, lq, rest)[0]
    assert bool(torch.isfinite(value).all()) and bool(torch.isfinite(torch.autograd.grad(value.sum(), a)[0]).all())
    assert float(distill.lm_head_distill(a, w, labels, ids, lq, rest, reverse=1.0)[0][0].detach()) == math.inf
