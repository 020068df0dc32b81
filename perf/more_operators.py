"""What the operators around a language model's output distribution are measured on: tokens drawn from logits with given random numbers
(temperature, top-k, top-p, min-p), the most likely tokens of rows of logits with their log-probabilities and what is left beside them,
and distillation from a teacher's most likely tokens through the output projection, with its gradients.

A draw.  Of a row of logits l at temperature T a token stays if ``l >= `` the ``top_k``-th largest logit, if ``exp((l - max) / T) >= min_p``,
and if the mass of the strictly larger ones among those that stayed so far is below ``top_p`` of theirs.  The drawn token is the first, in
the order of the vocabulary, up to which (itself included) the mass of what stayed is above ``u`` of the whole; at ``T <= 0`` it is the
first of the largest.  Its log-probability is that of the unrestricted row.

Most likely tokens: the ``k`` largest logits of a row, largest first, the lowest index first where they are equal, their log-probabilities
and the logarithm of the mass of all others.

Distillation.  A row has the teacher's probabilities q of K tokens (entries of -1 are none) and, where it is given, of all others together;
p are the student's, of the logits ``hidden @ weight^T * inv_temperature``.  With KL over these K (+ 1) classes the row's divergence is
``(1 - reverse) KL(q, p) + reverse KL(p, q)``.  Its gradients with respect to hidden states and weight are taken for given upstream
gradients of the rows.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` / ``run`` make and take one pass, ``exact`` is
the same pass in 64 bits, ``work`` the bytes and operations that a pass cannot do without.
"""
import math

import torch

own = False

SETTINGS = ("plain", "min_p", "top_p", "mixed")
VOCABULARIES = (32000, 151936, 151936, 248320)


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    def draws(name, rows, vocab, settings, dtype="float32", spare=0):
        return {"name": name, "kind": "draw", "rows": rows, "vocab": vocab, "settings": settings, "dtype": dtype, "spare": spare}

    def top(name, rows, vocab, k, dtype="float32", spare=0):
        return {"name": name, "kind": "top", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype, "spare": spare}

    def distill(name, rows, vocab, hidden, k, rest, reverse):
        return {"name": name, "kind": "distill", "rows": rows, "vocab": vocab, "hidden": hidden, "k": k, "rest": rest, "reverse": reverse}

    return [
        # one prompt, one answer: latency of a decode step's last part
        draws("draw-one", 1, 151936, "min_p"),
        # a decode step of the GRPO benchmark's rollouts, from the whole distribution
        draws("draw-rollouts", 128, 151936, "plain"),
        # the same with the nucleus that an evaluation asks for
        draws("draw-nucleus", 128, 151936, "top_p"),
        # requests of several users in one batch: each row its own settings, some greedy, logits of a padded buffer in 16 bits
        draws("draw-mixed", 41, 32000, "mixed", "bfloat16", 8),
        # the teacher's answer for one completion, a small model, an odd number of rows
        top("top-completion", 333, 32000, 20),
        # a chunk of rows of a scored batch
        top("top-chunk", 2048, 151936, 64),
        # the widest vocabulary, logits in 16 bits: many of them equal
        top("top-wide", 256, 248320, 128, "bfloat16"),
        # the smallest student, few rows: the weight is all there is to read
        distill("distill-few", 37, 32000, 256, 8, False, 0.0),
        # responses of a micro-batch, the teacher's top tokens alone
        distill("distill-forward", 549, 151936, 1024, 20, False, 0.0),
        # a student's own rollouts: towards the modes of the teacher
        distill("distill-reverse", 1500, 151936, 2048, 32, True, 1.0),
        # a chunk of 4096 rows of the benchmark's model, both directions
        distill("distill-chunk", 4096, 151936, 2560, 64, True, 0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("draw", "draw", "top", "top", "distill"))
    while True:
        vocab = rng.choice(VOCABULARIES + (rng.randint(1000, 160000),))
        if kind == "draw":
            c = {"kind": kind, "rows": _log(rng, 1, 256), "vocab": vocab, "settings": rng.choice(SETTINGS)}
        elif kind == "top":
            c = {"kind": kind, "rows": _log(rng, 1, 4096), "vocab": vocab, "k": _log(rng, 1, 256)}
        else:
            c = {"kind": kind, "rows": _log(rng, 1, 4096), "vocab": vocab // 8 * 8, "hidden": 64 * rng.randint(2, 40), "k": _log(rng, 1, 128),
                 "rest": rng.random() < 0.6, "reverse": rng.choice((0.0, 0.0, 0.25, 0.5, 1.0))}
        if kind != "distill":
            c.update(dtype=rng.choice(("float32", "float32", "bfloat16")), spare=rng.choice((0, 0, 1, 64)))
        if c["rows"] * c["vocab"] * (c["hidden"] / 2560 if kind == "distill" else 2) <= 4096 * 151936:
            return c


# ------------------------------------------------------------------------------------------------- data
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 1)


def _logits(g, rows, vocab, dtype, spare):
    """Rows in which a few tokens stand out, of some rows more and of some less, in a buffer with `spare` columns behind them."""
    x = torch.empty((rows, vocab + spare), device="cuda", dtype=getattr(torch, dtype))
    n = min(64, vocab // 4)
    for r0 in range(0, rows, 512):
        r = min(512, rows - r0)
        z = 2 * torch.randn((r, vocab + spare), device="cuda", generator=g)
        ids = torch.randint(vocab, (r, n), device="cuda", generator=g)
        height = 8 + 9 * torch.rand((r, 1), device="cuda", generator=g)
        boost = height - 2.5 * torch.log1p(torch.arange(n, device="cuda")) + torch.randn((r, n), device="cuda", generator=g)
        x[r0:r0 + r] = z.scatter_reduce(1, ids, boost, "amax")               # of a token that is named twice the larger one
    return x[:, :vocab]


def _settings(g, rows, kind):
    """Temperature, top-k, top-p and min-p of every row."""
    f = lambda v: torch.full((rows,), v, device="cuda")                                        # noqa: E731
    t, k, p, m = f(1.0), torch.zeros(rows, device="cuda", dtype=torch.int32), f(1.0), f(0.0)
    if kind == "min_p":
        t, m = f(0.8), f(0.05)
    elif kind == "top_p":
        t, p = f(0.7), f(0.95)
    elif kind == "mixed":
        pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(len(v), (rows,), device="cuda", generator=g)]     # noqa: E731
        t, k, p, m = pick(0.0, 0.6, 0.8, 1.0, 1.3), pick(0, 0, 20, 50, 400).to(torch.int32), pick(1.0, 0.8, 0.95, 0.99), pick(0.0, 0.0, 0.02, 0.1)
    return t, k, p, m


def prepare(case, seed):
    g, N, V = _gen(seed), case["rows"], case["vocab"]
    s = {"kind": case["kind"]}
    if case["kind"] == "distill":
        H, K = case["hidden"], case["k"]
        w = torch.randn((V, H), device="cuda", generator=g)
        s["weight"] = (w * (1.5 / math.sqrt(H))).to(torch.bfloat16)
        # a few tokens stand out in every row
        ids = torch.randint(V, (N, 8), device="cuda", generator=g)
        strength = (4 + 8 * torch.rand((N, 8), device="cuda", generator=g)) * torch.tensor([1, .8, .7, .6, .5, .4, .4, .3], device="cuda")
        h = torch.randn((N, H), device="cuda", generator=g) + torch.einsum("nk,nkh->nh", strength / (1.5 * math.sqrt(H)), w[ids])
        del w
        s["hidden"] = h.to(torch.bfloat16)
        s["labels"] = ids[:, 0]
        s["ids"] = torch.empty((N, K), device="cuda", dtype=torch.int32)
        s["logprobs"] = torch.empty((N, K), device="cuda")
        rest = torch.empty(N, device="cuda")
        for r0 in range(0, N, 1024):                   # the teacher: the student's logits, disturbed
            z = (s["hidden"][r0:r0 + 1024] @ s["weight"].t()).float()
            z += 1.5 * torch.randn(z.shape, device="cuda", generator=g)
            best, at = z.topk(K, dim=-1)
            lse = torch.logsumexp(z, -1, keepdim=True)
            s["ids"][r0:r0 + 1024], s["logprobs"][r0:r0 + 1024] = at.to(torch.int32), best - lse
            rest[r0:r0 + 1024] = torch.logsumexp(z.scatter(1, at, -math.inf), -1) - lse[:, 0]
        s["ids"][torch.rand((N, K), device="cuda", generator=g) < 0.02] = -1                 # entries that are none
        s["rest"] = rest if case["rest"] else None
        s["reverse"] = case["reverse"]
        s["inv_temperature"] = 1.0
        s["grad"] = torch.rand(N, device="cuda", generator=g) / N
        return s
    s["logits"] = _logits(g, N, V, case["dtype"], case["spare"])
    if case["kind"] == "top":
        s["k"] = case["k"]
        return s
    s["temperature"], s["top_k"], s["top_p"], s["min_p"] = _settings(g, N, case["settings"])
    s["u"] = torch.rand(N, device="cuda", generator=g)
    return s


# ------------------------------------------------------------------------------------------------- the plain forms
def _first_of_equal(x):
    """For rows in falling order: where the run of equal values begins that each one belongs to."""
    return torch.searchsorted(-x, -x, right=False)


def _plain_draw(s):
    z = s["logits"].double()                       # decided next to borders: 64 bits
    V = z.shape[1]
    at = torch.arange(V, device=z.device)
    greedy = ~(s["temperature"] > 0)
    T = torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    most = z.amax(-1, keepdim=True)
    x = (z - most) / T
    full = torch.exp(x)
    k = s["top_k"].long()
    k = torch.where((k > 0) & (k < V), k, V)[:, None]
    order = torch.sort(z, dim=-1, descending=True).values
    stays = (z >= order.gather(1, k - 1)) & (full >= s["min_p"].double()[:, None])
    mass = torch.where(stays, full, 0.0)
    # mass of the strictly larger ones, by rank
    weight = torch.exp((order - most) / T)
    weight = torch.where((order >= order.gather(1, k - 1)) & (weight >= s["min_p"].double()[:, None]), weight, 0.0)
    run = torch.cumsum(weight, -1)
    first = _first_of_equal(order)
    before = torch.where(first > 0, run.gather(1, (first - 1).clamp_min(0)), 0.0)
    p = s["top_p"].double()[:, None]
    last = ((before < p * run[:, -1:]) | (p >= 1)).sum(-1, keepdim=True)         # falling order: the first ones stay
    mass = torch.where(z >= order.gather(1, last.clamp_min(1) - 1), mass, 0.0)
    run = torch.cumsum(mass, -1)
    token = (run <= s["u"].double()[:, None] * run[:, -1:]).sum(-1)
    token = torch.minimum(token, torch.where(mass > 0, at, 0).amax(-1))
    token = torch.where(greedy, torch.where(z == most, at, V).amin(-1), token)
    logprob = x.gather(1, token[:, None])[:, 0] - torch.log(full.sum(-1))
    return token.to(torch.int32), logprob.float()


def _plain_top(s):
    z, k = s["logits"].float(), s["k"]
    order, at = torch.sort(z, dim=-1, descending=True, stable=True)
    e = torch.exp(order - order[:, :1])
    lse = order[:, :1] + torch.log(e.sum(-1, keepdim=True))
    left = order[:, k:k + 1] + torch.log(torch.exp(order[:, k:] - order[:, k:k + 1]).sum(-1, keepdim=True))
    named = torch.exp(order[:, :k] - lse).sum(-1)               # next to a logarithm of 1 its difference from 1 says more
    rest = torch.where(named < 0.5, torch.log1p(-named), (left - lse)[:, 0])
    return order[:, :k] - lse, at[:, :k].to(torch.int32), rest


def _times(x, y):
    """x y, nothing where x is nothing."""
    return torch.where(x > 0, x * y, 0.0)


def _plain_distill(s):
    h, w = s["hidden"].float(), s["weight"].float()
    V, it, b, rest = w.shape[0], s["inv_temperature"], s["reverse"], s["rest"]
    z = torch.nn.functional.pad(h @ w.t() * it, (0, 1), value=-math.inf)          # a last column for the entries that are none
    there = s["ids"] >= 0
    ids = torch.where(there, s["ids"], V).long()
    zk = z.gather(1, ids)
    logit = z.gather(1, s["labels"][:, None])[:, 0]
    most = z.amax(-1, keepdim=True)
    e = torch.exp(z - most)
    lse = most + torch.log(e.sum(-1, keepdim=True))
    left = torch.log(e.scatter(1, ids, 0.0).sum(-1, keepdim=True)) + most - lse
    del e
    lp, lq = zk - lse, torch.where(there, s["logprobs"], -math.inf)
    p, q = torch.exp(lp), torch.exp(lq)
    F = _times(q, lq - lp).sum(-1)
    R = _times(p, lp - lq).sum(-1)
    Q, E = q.sum(-1), _times(p, lp - lq + 1).sum(-1)
    on_rest = 0.0
    if rest is not None:
        pr, qr = torch.exp(left[:, 0]), torch.exp(rest)
        F, R, Q = F + _times(qr, rest - left[:, 0]), R + _times(pr, left[:, 0] - rest), Q + qr
        E = E + _times(pr, left[:, 0] - rest + 1)
        on_rest = -(1 - b) * qr / pr
        if b:
            on_rest = on_rest + b * (left[:, 0] - rest + 1)
    coefficient = (1 - b) * Q + on_rest
    special = (1 - b) * (p * Q[:, None] - q)
    if b:
        coefficient = coefficient - b * E
        special = special + b * _times(p, lp - lq + 1 - E[:, None])
    d = torch.exp(z - lse) * coefficient[:, None]
    del z
    d = (d.scatter(1, ids, special) * (s["grad"] * it)[:, None])[:, :V]
    value = (1 - b) * F + b * R if b else F
    return value, logit - lse[:, 0], (d @ w).to(s["hidden"].dtype), (d.t() @ h).to(s["weight"].dtype)


def run(s):
    if own:
        from arctic_platform_b200.ops import distill, logprob, sampling
        if s["kind"] == "draw":
            return sampling.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        if s["kind"] == "top":
            return logprob.top_logprobs(s["logits"], s["k"])
        h, w = s["hidden"].detach().requires_grad_(True), s["weight"].detach().requires_grad_(True)
        value, lp, _ = distill.lm_head_distill(h, w, s["labels"], s["ids"], s["logprobs"], s["rest"], s["inv_temperature"], s["reverse"],
                                               with_entropy=False)
        dh, dw = torch.autograd.grad(value, (h, w), s["grad"])
        return value.detach(), lp.detach(), dh, dw
    if s["kind"] == "draw":
        return _plain_draw(s)
    if s["kind"] == "top":
        return _plain_top(s)
    return _plain_distill(s)


# ------------------------------------------------------------------------------------------------- 64 bits
def _exact_draw(s):
    """Row by row: what stays, by a sorted walk; the draw by a search in the running mass."""
    out = []
    for r in range(s["logits"].shape[0]):
        z = s["logits"][r].double()
        T, k, p, m, u = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        if T <= 0:
            out.append(z.max() - torch.logsumexp(z, 0))
            continue
        z = z / T
        keep = torch.ones_like(z, dtype=torch.bool)
        if 0 < k < len(z):
            keep &= z >= z.topk(int(k)).values[-1]
        if m > 0:
            keep &= z - z.max() >= math.log(m)
        mass = torch.where(keep, torch.exp(z - z.max()), 0.0)
        if p < 1:
            value, back = torch.unique(z, return_inverse=True)                    # rising
            per = torch.zeros_like(value).index_add_(0, back, mass)
            larger = per.flip(0).cumsum(0).flip(0) - per
            mass = torch.where((larger < p * per.sum())[back], mass, 0.0)
        run = mass.cumsum(0)
        out.append(z[torch.searchsorted(run, u * run[-1:], right=True)[0].clamp_max(len(z) - 1)] - torch.logsumexp(z, 0))
    return None, torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "draw":
        return _exact_draw(s)
    N, V, parts = case["rows"], case["vocab"], []
    if case["kind"] == "top":
        for r0 in range(0, N, 128):
            z = s["logits"][r0:r0 + 128].double()
            value, at = z.topk(case["k"], -1)
            lse = torch.logsumexp(z, -1)
            parts.append((value - lse[:, None], torch.logsumexp(z.scatter(1, at, -math.inf), -1) - lse))
        return torch.cat([p[0] for p in parts]), None, torch.cat([p[1] for p in parts])
    w = s["weight"].double()
    dw, b = torch.zeros_like(w), case["reverse"]
    for r0 in range(0, N, 512):
        h = s["hidden"][r0:r0 + 512].double()
        n = len(h)
        lp = torch.log_softmax(h @ w.t() * s["inv_temperature"], -1)
        ids, there = s["ids"][r0:r0 + n].long().clamp_min(0), s["ids"][r0:r0 + n] >= 0
        lq = s["logprobs"][r0:r0 + n].double()
        # class of every token: its entry, or the one of all others
        classes = torch.full_like(lp, case["k"], dtype=torch.long)
        row = torch.arange(n, device="cuda")[:, None].expand_as(ids)[there]
        entry = torch.arange(case["k"], device="cuda").expand_as(ids)[there]
        classes[row, ids[there]] = entry
        named = torch.where(there, lp.gather(1, ids), -math.inf)
        others = torch.logsumexp(torch.where(classes == case["k"], lp, -math.inf), -1, keepdim=True)
        P = torch.cat([named, others], -1)
        L = torch.cat([torch.where(there, lq, 0.0), s["rest"][r0:r0 + n, None].double() if case["rest"] else torch.zeros_like(others)], -1)
        counts = torch.cat([there, torch.full_like(others, case["rest"], dtype=torch.bool)], -1)
        prob, q = torch.where(counts, P.exp(), 0.0), torch.where(counts, L.exp(), 0.0)
        gap = torch.where(counts, L - P, 0.0)
        value = (1 - b) * (q * gap).sum(-1) - b * (prob * gap).sum(-1)
        # d value / d log P of every class, and of the tokens: through log P = logsumexp of the class's tokens
        by_class = -(1 - b) * q + b * prob * (1 - gap)
        inside = torch.exp(lp - P.gather(1, classes))
        d = by_class.gather(1, classes) * inside - by_class.sum(-1, keepdim=True) * lp.exp()
        d *= s["grad"][r0:r0 + n, None].double() * s["inv_temperature"]
        parts.append((value, lp.gather(1, s["labels"][r0:r0 + n, None])[:, 0], d @ w))
        dw += d.t() @ h
    return tuple(torch.cat(x) for x in zip(*parts)) + (dw,)


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    N, V = case["rows"], case["vocab"]
    if case["kind"] == "distill":
        H, K = case["hidden"], case["k"]
        return {"bytes": float(4 * (V * H + N * H) + N * (8 * K + 16 + 4 * case["rest"])), "flops": 6.0 * N * V * H}
    size = 4 if case["dtype"] == "float32" else 2
    out = 8 * case["k"] + 4 if case["kind"] == "top" else 28
    return {"bytes": float(N * (V * size + out)), "flops": 2.0 * N * V}
