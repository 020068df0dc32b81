"""Distillation through the lm head on a GPU against the fp64 expression, values and gradients.

Logits: products are exact in fp32; the tensor cores' running sum of H terms is off by at most H 2^-23 of the sum of magnitudes S (which is
below 30 here), fp32 sums by less: ``ERR = 256 * 2^-23 * 30 < 1e-3``.  A log-probability is off by twice that, a divergence by at most
twice that per unit of mass, of which q and p have one each: 4 ERR.  d(logits) is rounded to bf16 (2^-8 of it, or less by half: finfo.eps
/ 2), and off by the probabilities' relative error of 2 ERR before; the products add fp32 rounding far below that, and the results are rounded to
bf16 again.  So a gradient's element is off by (2^-8 + 4 ERR) of its sum of magnitudes and 2^-8 of itself."""
import pytest
import torch

from arctic_platform_b200.ops import distill, logprob

pytestmark = pytest.mark.gpu
ERR = 1e-3


def make(N, V, H, K, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn((V, H), device="cuda", generator=g) * (1.2 / H ** 0.5)).bfloat16()
    h = torch.randn((N, H), device="cuda", generator=g).bfloat16()
    t = h.float() @ w.float().t() + torch.randn((N, V), device="cuda", generator=g)
    lq, ids, rest = logprob.top_logprobs_ref(t, K)
    labels = torch.randint(V, (N,), device="cuda", generator=g)
    labels[::3] = ids[::3, 0].long()                           # labels that are named, and others
    return h, w, labels, ids, lq, rest


def gradients(h, w, labels, ids, lq, rest, it, reverse, ups, entropy=True):
    """Values, gradients of hidden and weight, and their sums of magnitudes, in 64 bits."""
    z = (h.double() @ w.double().t()).requires_grad_(True)
    eye = torch.eye(w.shape[0], dtype=torch.float64, device="cuda")
    out = distill.distill_ref(z, eye, labels, ids, lq, rest, it, reverse, entropy, torch.float64)
    (d,) = torch.autograd.grad([o for o, u in zip(out, ups) if u is not None], z, [u.double() for u in ups if u is not None])
    return out, d @ w.double(), d.t() @ h.double(), d.abs() @ w.double().abs(), d.abs().t() @ h.double().abs()


def check(N, V, H, K, with_rest, reverse, it=1.0, entropy=True, ups=None, chunk=None, data=None, seed=0, roundings=1):
    h, w, labels, ids, lq, rest = data or make(N, V, H, K, seed)
    rest = rest if with_rest else None
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    if ups is None:
        ups = [torch.randn(N, device="cuda", generator=g) for _ in range(3)]
    if not entropy:
        ups[2] = None
    want, dh, dw, sh, sw = gradients(h, w, labels, ids, lq, rest, it, reverse, ups, entropy)
    hl, wl = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    got = distill.lm_head_distill(hl, wl, labels, ids, lq, rest, it, reverse, entropy, chunk)
    assert (got[2] is None) == (not entropy)
    scale = float(it.max()) if torch.is_tensor(it) else it
    for a, b in zip(got, want):
        if a is not None:
            torch.testing.assert_close(a.double(), b, rtol=2.0 ** -20, atol=4 * ERR * max(scale, 1))
    grads = torch.autograd.grad([o for o, u in zip(got, ups) if u is not None], (hl, wl), [u for u in ups if u is not None])
    for a, b, s in zip(grads, (dh, dw), (sh, sw)):
        off = (a.double() - b).abs()
        assert bool((off <= (roundings * 2.0 ** -8 + 4 * ERR * max(scale, 1)) * s + 2.0 ** -8 * b.abs() + 1e-12).all()), float((off / s.clamp_min(1e-9)).max())
    return got, grads


@pytest.mark.parametrize("N,V,H,K", [(1, 8, 8, 1), (5, 136, 64, 8), (37, 1000, 256, 20), (129, 2008, 128, 64), (300, 520, 72, 256), (260, 4096, 256, 3)])
@pytest.mark.parametrize("with_rest,reverse", [(False, 0.0), (True, 0.0), (True, 1.0), (False, 1.0), (True, 0.4)])
def test_values_and_gradients(N, V, H, K, with_rest, reverse):
    check(N, V, H, min(K, V), with_rest, reverse, seed=N)


@pytest.mark.parametrize("N,V,H,K", [(1, 8, 8, 1), (5, 136, 64, 8), (129, 2008, 128, 64), (300, 520, 72, 256), (260, 4096, 256, 3), (700, 392, 64, 5)])
@pytest.mark.parametrize("reverse", [0.0, 0.4])
def test_exponentials_kept_for_the_backward_pass(N, V, H, K, reverse, monkeypatch):
    """A probability is rounded to bf16 once more (and by the square of a rounding, which 2^-8 of its 4 ERR covers)."""
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: True)
    one = torch.linspace(-1, 1, N, device="cuda")
    more = {"roundings": 2, "seed": N}
    check(N, V, H, min(K, V), True, reverse, ups=[one, one.flip(0), None], **more)
    check(N, V, H, min(K, V), True, reverse, it=torch.linspace(0.3, 1.5, N, device="cuda"), ups=[one, None, None], chunk=256, **more)
    check(N, V, H, min(K, V), True, reverse, **more)           # an entropy's gradient too: formed from the logits again


def test_kept_exponentials_serve_two_backward_passes_and_one_is_chosen_by_size(monkeypatch):
    h, w, labels, ids, lq, rest = make(512, 131072, 64, 8, 11)         # from 2^26 on they are kept
    hl, wl = h.requires_grad_(True), w.requires_grad_(True)
    value = distill.lm_head_distill(hl, wl, labels, ids, lq, rest, reverse=0.5)[0].sum()
    kept = [t for t in value.grad_fn.next_functions[0][0].saved_tensors if t is not None and t.shape == (512, 131072)]
    assert len(kept) == 1 and kept[0].dtype == torch.bfloat16
    a = torch.autograd.grad(value, (hl, wl), retain_graph=True)
    b = torch.autograd.grad(value, (hl, wl))
    assert torch.equal(a[1], b[1])
    torch.testing.assert_close(a[0], b[0], rtol=2.0 ** -7, atol=1e-6)    # parts of the vocabulary add up in any order
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: False)
    c = torch.autograd.grad(distill.lm_head_distill(hl, wl, labels, ids, lq, rest, reverse=0.5)[0].sum(), (hl, wl))
    for x, y in zip(a, c):
        assert float((x.double() - y.double()).norm() / y.double().norm()) < 2.0 ** -7     # each once or twice off by 2^-8 and 2^-9 on average


def test_temperatures_and_no_entropy():
    check(40, 640, 128, 16, True, 0.3, it=0.7)
    check(40, 640, 128, 16, True, 0.3, it=torch.linspace(0.3, 1.5, 40, device="cuda"))
    check(40, 640, 128, 16, True, 0.3, entropy=False)


def test_one_output_at_a_time_and_chunks():
    one = torch.ones(70, device="cuda")
    for ups in ([one, None, None], [None, one, None], [None, None, one]):
        check(70, 776, 128, 9, True, 0.5, ups=list(ups))
    a = check(600, 520, 64, 12, True, 0.5, chunk=256)[1]
    b = check(600, 520, 64, 12, True, 0.5)[1]
    torch.testing.assert_close(a[0], b[0], rtol=2.0 ** -7, atol=1e-3)


def test_logprob_and_entropy_are_those_of_the_lm_head():
    h, w, labels, ids, lq, rest = make(200, 3000, 256, 32)
    _, lp, ent = distill.lm_head_distill(h, w, labels, ids, lq, rest)
    lp2, ent2 = logprob.lm_head_logprobs(h, w, labels)
    torch.testing.assert_close(lp, lp2, rtol=0, atol=4 * ERR)
    torch.testing.assert_close(ent, ent2, rtol=0, atol=8 * ERR)


@pytest.mark.parametrize("reverse", [0.0, 0.5])
@pytest.mark.parametrize("with_rest", [False, True])
def test_entries_that_name_nothing_or_name_again(with_rest, reverse):
    h, w, labels, ids, lq, rest = make(30, 400, 128, 10, 3)
    ids[0] = -1
    ids[1, 3:] = -1
    ids[2, 4] = ids[2, 9] = ids[2, 1]
    ids[3, 2] = 400
    ids[4, 0] = 2 ** 31 - 1
    ids[5, 5] = -2 ** 31
    ids[6] = ids[6, 0]
    if with_rest:
        rest = torch.where(torch.arange(30, device="cuda") == 0, torch.zeros_like(rest), rest)
    got, _ = check(30, 400, 128, 10, with_rest, reverse, data=(h, w, labels, ids, lq, rest))
    assert abs(float(got[0][0].detach())) < 4 * ERR
    far = ids.long()
    far[7, 1] = 2 ** 32 + 5                                    # not 5
    lost = torch.where(far == 2 ** 32 + 5, -1, far)
    a = distill.lm_head_distill(h, w, labels, far, lq, rest if with_rest else None, reverse=reverse)[0]
    b = distill.lm_head_distill(h, w, labels, lost, lq, rest if with_rest else None, reverse=reverse)[0]
    assert torch.equal(a, b)


def test_classes_without_mass():
    h, w, labels, ids, lq, rest = make(12, 256, 64, 6, 4)
    inf = float("inf")
    lq[0, 2] = -inf                                            # the teacher gives a named token nothing
    rest[1] = -inf                                             # the named tokens are all it gives anything to
    check(12, 256, 64, 6, True, 0.0, data=(h, w, labels, ids, lq, rest))
    value, _, _ = distill.lm_head_distill(h, w, labels, ids, lq, rest, reverse=1.0)
    assert float(value[0]) == inf and float(value[1]) == inf and bool(torch.isfinite(value[2:]).all())
    # all tokens named: no others
    h, w, labels, ids, lq, rest = make(4, 64, 64, 64, 5)
    check(4, 64, 64, 64, True, 0.5, data=(h, w, labels, ids, lq, rest))
    # rows that infinite divergences are masked out of
    h, w, labels, ids, lq, rest = make(12, 256, 64, 6, 4)
    lq[3, 1] = -inf
    hl, wl = h.requires_grad_(True), w.requires_grad_(True)
    value = distill.lm_head_distill(hl, wl, labels, ids, lq, rest, reverse=1.0)[0]
    up = torch.ones_like(value)
    up[3] = 0
    dh, dw = torch.autograd.grad(value, (hl, wl), up)
    assert bool(torch.isfinite(dh).all()) and bool(torch.isfinite(dw).all()) and bool((dh[3] == 0).all())


def test_a_student_that_is_sure():
    """Nearly all mass on a named token: the others' mass comes from their own sum."""
    g = torch.Generator(device="cuda").manual_seed(6)
    w = (torch.randn((800, 64), device="cuda", generator=g) / 8).bfloat16()
    ids = torch.randint(800, (50, 5), device="cuda", generator=g)
    h = (10 * w[ids[:, 0]].float()).bfloat16()                 # the first named token is 10 nats above most
    lq = torch.log_softmax(torch.randn((50, 6), device="cuda", generator=g), -1)
    labels = ids[:, 0].clone()
    for reverse in (0.0, 0.5):
        check(50, 800, 64, 5, True, reverse, data=(h, w, labels, ids, lq[:, :5].contiguous(), lq[:, 5].contiguous()))


def test_gradients_accumulate_in_fp32_where_the_engine_keeps_them():
    h, w, labels, ids, lq, rest = make(40, 256, 64, 6, 7)
    want = gradients(h, w, labels, ids, lq, rest, 1.0, 0.0, [torch.ones(40, device="cuda"), None, None])
    hl, wl = h.requires_grad_(True), w.requires_grad_(True)
    wl.grad_f32 = torch.ones((256, 64), device="cuda")
    distill.lm_head_distill(hl, wl, labels, ids, lq, rest)[0].sum().backward()
    assert wl.grad is None
    off = (wl.grad_f32.double() - 1 - want[2]).abs()
    assert bool((off <= (2.0 ** -8 + 4 * ERR) * want[4] + 1e-6).all())
    # frozen weight, frozen student
    dh = torch.autograd.grad(distill.lm_head_distill(hl, w.detach(), labels, ids, lq, rest)[0].sum(), hl)[0]
    torch.testing.assert_close(dh, hl.grad)
    assert not distill.lm_head_distill(h.detach(), w.detach(), labels, ids, lq, rest)[0].requires_grad


def test_strides_streams_and_a_captured_forward():
    h, w, labels, ids, lq, rest = make(33, 512, 64, 7, 8)
    want = distill.lm_head_distill(h, w, labels, ids, lq, rest)[0]
    wide = torch.zeros((33, 200), device="cuda", dtype=torch.bfloat16)
    for c in (0, 3, 8):
        wide[:, c:c + 64] = h
        assert torch.equal(distill.lm_head_distill(wide[:, c:c + 64], w, labels, ids, lq, rest)[0], want)
    assert torch.equal(distill.lm_head_distill(h, w, labels, ids.t().contiguous().t(), lq.double(), rest)[0], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = distill.lm_head_distill(h, w, labels, ids, lq, rest)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    lab32 = labels.to(torch.int32)
    with torch.cuda.graph(graph):
        got = distill.lm_head_distill(h, w, lab32, ids, lq, rest)[0]
    graph.replay()
    assert torch.equal(got, want)


def test_expanded_rows_and_overlapping_ones():
    h, w, labels, ids, lq, rest = make(9, 256, 64, 6, 12)
    one = h[:1].expand(9, 64)
    assert one.stride(0) == 0
    want = distill.lm_head_distill(one.contiguous(), w, labels, ids, lq, rest)[0]
    hl = h[:1].detach().requires_grad_(True)
    got = distill.lm_head_distill(hl.expand(9, 64), w, labels, ids, lq, rest)[0]
    assert torch.equal(got, want)
    (d,) = torch.autograd.grad(got.sum(), hl)
    each = [torch.autograd.grad(distill.lm_head_distill(x, w, labels[i:i + 1], ids[i:i + 1], lq[i:i + 1], rest[i:i + 1])[0].sum(), x)[0]
            for i in range(9) for x in [h[:1].detach().requires_grad_(True)]]
    many = torch.stack(each).double()
    # nine gradients in bf16 each (2^-8 twice: d(logits) and the row) add up in bf16
    assert bool(((d.double() - many.sum(0)).abs() <= 12 * 2.0 ** -8 * many.abs().sum(0) + 1e-2 * many.abs().amax()).all())
    again = lq[:1].expand(9, 6)
    a = distill.lm_head_distill(h, w, labels, ids[:1].expand(9, 6), again, rest[:1].expand(9))[0]
    b = distill.lm_head_distill(h, w, labels, ids[:1].expand(9, 6).contiguous(), again.contiguous(), rest[:1].expand(9).contiguous())[0]
    assert torch.equal(a, b)
    with pytest.raises(ValueError):
        distill.lm_head_distill(h, w[:1].expand(256, 64), labels, ids, lq, rest)


@pytest.mark.parametrize("keep", [False, True])
def test_a_captured_forward_and_backward_pass(keep, monkeypatch):
    monkeypatch.setattr(distill, "_keep_pays", lambda *a: keep)
    h, w, labels, ids, lq, rest = make(300, 520, 64, 7, 13)
    lab32, up = labels.to(torch.int32), torch.linspace(-1, 1, 300, device="cuda")

    def run(hl, wl):
        value, lp, _ = distill.lm_head_distill(hl, wl, lab32, ids, lq, rest, reverse=0.5)
        return torch.autograd.grad([value, lp], (hl, wl), [up, up])

    want = run(h.clone().requires_grad_(True), w.clone().requires_grad_(True))
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(hl, wl)
    for _ in range(2):
        for g in got:
            g.zero_()
        graph.replay()
        assert torch.equal(got[1], want[1])
        torch.testing.assert_close(got[0], want[0], rtol=2.0 ** -7, atol=1e-6)     # parts of the vocabulary add up in any order
    with torch.no_grad():
        hl.copy_(h.flip(0))
    graph.replay()
    new = run(h.flip(0).clone().requires_grad_(True), w.clone().requires_grad_(True))
    assert torch.equal(got[1], new[1]) and not torch.equal(got[1], want[1])


def test_two_passes_on_two_streams_at_once():
    data = [make(200, 1000, 128, 9, s) for s in (14, 15)]

    def run(d):
        h, w, labels, ids, lq, rest = d
        hl, wl = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        return torch.autograd.grad(distill.lm_head_distill(hl, wl, labels, ids, lq, rest, reverse=0.3)[0].sum(), (hl, wl))

    want = [run(d) for d in data]
    sides = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, d in enumerate(data):
            with torch.cuda.stream(sides[i]):
                got[i].append(run(d))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g[1], want[i][1])
            torch.testing.assert_close(g[0], want[i][0], rtol=2.0 ** -7, atol=1e-5)


def test_refusals():
    h, w, labels, ids, lq, rest = make(8, 64, 64, 4, 9)
    f = distill.lm_head_distill
    for bad in (lambda: f(h[:, :60], w[:, :60], labels, ids, lq), lambda: f(h, w[:60], labels, ids, lq), lambda: f(h.float(), w.float(), labels, ids, lq),
                lambda: f(h, w, labels[:7], ids, lq), lambda: f(h, w, labels, ids, lq[:, :3]), lambda: f(h, w, labels, ids.float(), lq),
                lambda: f(h, w, labels, ids, lq, rest[:5]), lambda: f(h, w, labels, ids, lq, rest, reverse=1.5),
                lambda: f(h, w, labels, ids, lq, rest, reverse=-0.1), lambda: f(h, w, labels, ids.cpu(), lq),
                lambda: f(h, w, labels, torch.zeros((8, 257), device="cuda", dtype=torch.int32), torch.zeros((8, 257), device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    z = f(h[:0].requires_grad_(True), w.detach().requires_grad_(True), labels[:0], ids[:0], lq[:0], rest[:0])
    assert z[0].shape == (0,) and z[0].requires_grad
