"""What the operators of the 8-bit key/value cache are measured on: rows of keys and values quantised into the cache and read back,
attention of single query tokens over it, attention of chunks of tokens over it.

A cache block holds 16 tokens of one key head: 16 rows of D codes (e4m3) of the keys, 16 rows of the values, then 32 bytes of
exponents.  A row's values are ``code * 2^(byte - 127)``; the byte of token t is at ``4 (t % 8) + t // 8`` for its key, two further on
for its value.  The exponent is the least one, of -100 to 119, with which the row's largest magnitude is no more than 448, the largest e4m3 number.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` / ``run`` make and take one pass, ``exact`` is
the same pass in 64 bits, ``work`` the bytes and operations that a pass cannot do without.
"""
import math
import random

import torch

own = False

PAGE = 16
LEAST, MOST = -100, 119              # exponents of a row
HEADS = ((16, 8), (32, 8), (32, 4), (64, 8), (4, 2), (8, 8), (14, 2), (16, 1), (5, 1))      # query heads, key heads


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    def rows(kind, name, tokens, kv_heads, dim=128, dtype="bfloat16"):
        return {"name": name, "kind": kind, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "dtype": dtype}

    def decode(name, batch, length, even, heads, kv_heads, dim=128):
        return {"name": name, "kind": "decode", "batch": batch, "length": length, "even": even, "heads": heads,
                "kv_heads": kv_heads, "dim": dim}

    def chunk(name, batch, new, length, even, heads, kv_heads, dim=128):
        return {"name": name, "kind": "chunk", "batch": batch, "new": new, "length": length, "even": even, "heads": heads,
                "kv_heads": kv_heads, "dim": dim}

    return [
        # one decode step of the GRPO benchmark's rollouts: a new token for each of 128 sequences
        rows("store", "store-step", 128, 8),
        # its 8 prompts of 2048 tokens
        rows("store", "store-prompts", 16384, 8),
        # the small test model in fp32, an odd number of rows
        rows("store", "store-odd", 1001, 2, 64, "float32"),
        # a header of 333 tokens that a new prompt is to attend to
        rows("read", "read-header", 333, 8),
        # the longest prompt and response of the recipes
        rows("read", "read-long", 36864, 4),
        # one prompt, one answer: latency of a decode step
        decode("decode-one", 1, 384, True, 32, 8),
        # evaluation: distinct prompts of uneven length
        decode("decode-ragged", 41, 1500, False, 16, 8),
        # the rollouts of the benchmark in the middle of their responses
        decode("decode-rollouts", 128, 4096, False, 32, 8),
        # long context, few sequences
        decode("decode-long", 2, 36864, True, 32, 4),
        # a draft of 5 tokens is checked for each of 16 sequences
        chunk("chunk-drafts", 16, 5, 1500, False, 32, 8),
        # a conversation goes on: 512 tokens behind 16384
        chunk("chunk-turn", 1, 512, 16896, True, 32, 8),
        # whole prompts of uneven length over what they have just stored
        chunk("chunk-prompts", 4, 4096, 4096, False, 32, 8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("store", "read", "decode", "decode", "chunk", "chunk"))
    dim = rng.choice((64, 128, 128))
    heads, kv_heads = rng.choice(HEADS)
    while True:
        if kind in ("store", "read"):
            c = {"kind": kind, "tokens": _log(rng, 1, 36864), "kv_heads": kv_heads, "dim": dim,
                 "dtype": rng.choice(("bfloat16", "bfloat16", "float32")) if kind == "store" else "bfloat16"}
            return c if c["tokens"] * kv_heads * dim <= 16384 * 8 * 128 else dict(c, tokens=rng.randint(1, 2000))
        c = {"kind": kind, "batch": _log(rng, 1, 128), "length": _log(rng, 1, 36864), "even": rng.random() < 0.3, "heads": heads,
             "kv_heads": kv_heads, "dim": dim}
        if kind == "chunk":
            c = {"kind": kind, "batch": _log(rng, 1, 24), "new": _log(rng, 2, 2048), **{k: c[k] for k in list(c)[2:]}}
            c["new"] = min(c["new"], c["length"])
        if work(c)["flops"] <= 1e11 and work(c)["bytes"] <= 8e8 and c["batch"] * c["length"] <= 400000:
            return c


# ------------------------------------------------------------------------------------------------- sizes and data
def _lengths(case):
    """Tokens in the cache and, for chunks, how many of them are new: uneven, the same for every seed."""
    rng = random.Random("%d %d" % (case["batch"], case["length"]))
    lengths = [case["length"] if case["even"] else rng.randint(max(1, case["length"] // 3), case["length"]) for _ in range(case["batch"])]
    if case["batch"] > 8 and not case["even"]:
        lengths[3] = 0 if case["kind"] == "decode" else 1       # an idle slot; a sequence that has just begun
    new = [min(n, case["new"]) if case["even"] or case["new"] < 16 else min(n, rng.randint(case["new"] // 2, case["new"])) for n in lengths] \
        if case["kind"] == "chunk" else [1] * len(lengths)
    return lengths, new


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 1)


def _rows(g, n, heads, dim, channel, spread):
    """Keys or values of n tokens: channels of unlike size, tokens of unlike size."""
    x = torch.randn((n, heads, dim), device="cuda", generator=g)
    return x * channel * torch.exp(spread * torch.randn((n, heads, 1), device="cuda", generator=g))


def _scales(g, heads, dim):
    """Sizes of the channels: a few of the keys' stand out; the scores then have a deviation of about 1.5."""
    k = torch.exp(0.5 * torch.randn((heads, dim), device="cuda", generator=g))
    k[:, 3::29] *= 6
    return 1.5 * k / k.square().mean(-1, keepdim=True).sqrt(), torch.exp(0.3 * torch.randn((heads, dim), device="cuda", generator=g))


def _block(dim):
    return 2 * PAGE * dim + 2 * PAGE


def prepare(case, seed):
    g, H, D = _gen(seed), case["kv_heads"], case["dim"]
    ck, cv = _scales(g, H, D)
    s = {"dim": D, "kind": case["kind"]}
    if case["kind"] in ("store", "read"):
        T = case["tokens"]
        pages = -(-T // PAGE) + 5
        s["data"] = torch.zeros((pages, H, _block(D)), device="cuda", dtype=torch.uint8)
        slots = torch.randperm(pages, device="cuda", generator=g)[:-(-T // PAGE), None] * PAGE + torch.arange(PAGE, device="cuda")
        s["slots"] = slots.reshape(-1)[:T].to(torch.int32).contiguous()
        if T > 20:
            s["slots"][torch.randperm(T, device="cuda", generator=g)[:T // 20]] = -1       # rows of padding
        dt = getattr(torch, case["dtype"])
        # the columns of one projection, as a layer leaves them
        kv = torch.cat([_rows(g, T, H, D, ck, 0.3), _rows(g, T, H, D, cv, 0.5)], 1).to(dt)
        s["k"], s["v"] = kv[:, :H], kv[:, H:]
        if case["kind"] == "read":
            _store(s["data"], s["k"], s["v"], s["slots"])
    else:
        lengths, new = _lengths(case)
        n_pages = [-(-n // PAGE) for n in lengths]
        pages, wide = sum(n_pages) + 3, max(max(n_pages), 1)
        s["data"] = torch.empty((pages, H, _block(D)), device="cuda", dtype=torch.uint8)
        for p0 in range(0, pages, 4096):                      # in parts that need little memory
            n = min(4096, pages - p0)
            at = torch.arange(n * PAGE, device="cuda")
            _store(s["data"][p0:p0 + n], _rows(g, n * PAGE, H, D, ck, 0.3).bfloat16(), _rows(g, n * PAGE, H, D, cv, 0.5).bfloat16(), at)
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        first = [sum(n_pages[:i]) for i in range(len(n_pages))]
        index = torch.tensor(first, device="cuda")[:, None] + torch.arange(wide, device="cuda")
        there = torch.arange(wide, device="cuda") < torch.tensor(n_pages, device="cuda")[:, None]
        s["table"] = torch.where(there, order[index.clamp_max(pages - 1)], 0).to(torch.int32).contiguous()
        s["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
        s["new"] = torch.tensor(new, device="cuda", dtype=torch.int32)
        s["most_new"], s["rows"] = max(new), sum(new)
        q = torch.randn((sum(new), case["heads"], D), device="cuda", generator=g)
        s["q"] = q.to(torch.bfloat16)
    if own:
        from arctic_platform_b200.ops import kv_fp8
        s["cache"] = kv_fp8.Fp8KVCache(s["data"], D)
        if case["kind"] == "chunk":
            s["plan"] = kv_fp8.ChunkPlan.build(new, lengths, s["table"].cpu().numpy(), case["heads"], s["cache"])
    return s


# ------------------------------------------------------------------------------------------------- the plain forms
def _parts(data, dim):
    """Views of the blocks: codes ``[pages, heads, 2, 16, dim]`` (keys, values), exponents ``[pages, heads, 8, 2, 2]`` (token % 8, key or
    value, token // 8)."""
    n = 2 * PAGE * dim
    return data[..., :n].unflatten(-1, (2, PAGE, dim)), data[..., n:].unflatten(-1, (8, 2, 2))


def _quantise(x):
    """Rows of numbers to codes (as bytes) and exponents + 127."""
    x = x.float()
    most = x.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(most)                   # most = mantissa * 2^exponent, mantissa from 1/2 on; 448 = 0.875 * 2^9
    e = torch.where(most > 0, exponent - 9 + (mantissa > 0.875), LEAST).clamp(LEAST, MOST)
    codes = torch.ldexp(x, -e).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).squeeze(-1).to(torch.uint8)


def _store(data, k, v, slots):
    codes, ex = _parts(data, k.shape[-1])
    keep = (slots >= 0).nonzero()[:, 0]
    at = slots[keep].long()
    page, t = at // PAGE, at % PAGE
    codes[page, :, :, t], ex[page, :, t % 8, :, t // 8] = _quantise(torch.stack((k, v), 2)[keep])


def _values(codes, byte):
    """Codes ``[..., dim]`` and exponent bytes ``[...]`` to fp32."""
    return torch.ldexp(codes.contiguous().view(torch.float8_e4m3fn).float(), (byte.int() - 127)[..., None])


def _read(data, slots, dim):
    codes, ex = _parts(data, dim)
    at = slots.long().clamp_min(0)
    page, t = at // PAGE, at % PAGE
    x = _values(codes[page, :, :, t], ex[page, :, t % 8, :, t // 8])
    return (x * (slots >= 0)[:, None, None, None]).to(torch.bfloat16).unbind(2)


def _context(data, table, dim):
    """Keys and values of whole page lists: two of ``[batch, heads, pages * 16, dim]`` in fp32."""
    codes, ex = _parts(data, dim)
    byte = ex.permute(0, 1, 3, 4, 2).flatten(-2)               # [pages, heads, 2, 16]
    x = _values(codes[table.long()], byte[table.long()])       # [batch, pages, heads, 2, 16, dim]
    return x.permute(3, 0, 2, 1, 4, 5).flatten(3, 4).unbind(0)


def _attend(q, k, v, visible):
    """``q [batch, kv heads, rows, dim]`` fp32; ``visible [batch, 1, rows, tokens]``; rows that see nothing are zeros."""
    s = (q @ k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    s = s.masked_fill(~visible, float("-inf"))
    most = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(most == float("-inf"), 0, most))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total > 0, total, 1)


def run(s):
    if own:
        from arctic_platform_b200.ops import kv_fp8
        if s["kind"] == "store":
            kv_fp8.write(s["k"], s["v"], s["slots"], s["cache"])
        if s["kind"] in ("store", "read"):
            return kv_fp8.read(s["cache"], s["slots"])
        if s["kind"] == "decode":
            return kv_fp8.decode_attention(s["q"], s["cache"], s["table"], s["lengths"])
        return kv_fp8.chunk_attention(s["q"], s["cache"], s["plan"])
    D = s["dim"]
    if s["kind"] == "store":
        _store(s["data"], s["k"], s["v"], s["slots"])
    if s["kind"] in ("store", "read"):
        return _read(s["data"], s["slots"], D)
    q, H = s["q"].float(), s["data"].shape[1]
    R = q.shape[1] // H
    k, v = _context(s["data"], s["table"], D)
    tokens = torch.arange(k.shape[2], device=q.device)
    B, N, lengths = len(s["lengths"]), s["most_new"], s["lengths"].long()
    # the rows of every sequence side by side, padded to the longest
    new = s["new"].long()
    first = torch.cumsum(new, 0) - new
    i = torch.arange(N, device=q.device)
    at = (first[:, None] + torch.minimum(i, new[:, None] - 1)).clamp_min(0)               # [B, N]
    x = q[at].unflatten(2, (H, R)).permute(0, 2, 1, 3, 4).reshape(B, H, N * R, D)
    last = lengths[:, None] - new[:, None] + i if s["kind"] == "chunk" else lengths[:, None] - 1        # position of each row
    visible = tokens <= last[..., None]
    o = _attend(x, k, v, visible.repeat_interleave(R, 1)[:, None])
    o = o.reshape(B, H, N, R, D).permute(0, 2, 1, 3, 4).reshape(B, N, H * R, D)
    return o[i < new[:, None]].to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------- 64 bits
def _e4m3(x):
    """The nearest e4m3 numbers, even ones at ties."""
    _, e = torch.frexp(x.abs())                              # |x| = m 2^e, 1/2 <= m < 1
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return torch.round(x / step) * step


def _block_values(blocks, dim, which):
    """Values of the blocks ``[n, heads, bytes]`` in 64 bits: ``[n, heads, 16, dim]``; which: 0 keys, 1 values."""
    b = blocks.int()
    c = b[..., which * PAGE * dim:(which + 1) * PAGE * dim].unflatten(-1, (PAGE, dim))
    field, fraction = c % 128 // 8, (c % 8).double()
    size = torch.where(field > 0, (8 + fraction) * torch.exp2(field.double() - 10), fraction * 2.0 ** -9)
    t = torch.arange(PAGE, device=b.device)
    e = b[..., 2 * PAGE * dim:][..., 4 * (t % 8) + 2 * which + t // 8]
    return torch.where(c >= 128, -size, size) * torch.exp2(e.double() - 127)[..., None]


def exact(case, seed):
    if case["kind"] in ("decode", "chunk") and work(case)["flops"] > 6e11:
        return None
    s = prepare(case, seed)
    D = case["dim"]
    if case["kind"] == "store":
        out = []
        for x in (s["k"], s["v"]):
            x = x.double()
            most = x.abs().amax(-1, keepdim=True)
            e = torch.ceil(torch.log2(most / 448)).clamp(LEAST, MOST)
            e = torch.where(torch.exp2(e - 1) * 448 >= most, e - 1, e)           # a logarithm that fell on the wrong side of a whole number
            e = torch.where(torch.exp2(e) * 448 < most, e + 1, e)
            out.append(_e4m3(x / torch.exp2(e)) * torch.exp2(e) * (s["slots"] >= 0)[:, None, None])
        return tuple(out)
    if case["kind"] == "read":
        at = s["slots"].long().clamp_min(0)
        return tuple(_block_values(s["data"][at // PAGE], D, w)[torch.arange(len(at), device="cuda"), :, at % PAGE]
                     * (s["slots"] >= 0)[:, None, None] for w in (0, 1))
    out, row = [], 0
    R = case["heads"] // case["kv_heads"]
    for b, (n, m) in enumerate(zip(*_lengths(case))):
        q = s["q"][row:row + m].double()
        row += m
        if n == 0:
            out.append(torch.zeros_like(q))
            continue
        blocks = s["data"][s["table"][b, :-(-n // PAGE)].long()]
        o = torch.empty_like(q)
        for h in range(case["kv_heads"]):
            k, v = (_block_values(blocks[:, h:h + 1], D, w)[:, 0].reshape(-1, D)[:n] for w in (0, 1))
            for m0 in range(0, m, 256):
                x = q[m0:m0 + 256, h * R:(h + 1) * R]
                sc = torch.einsum("ird,td->irt", x, k) * D ** -0.5
                at = torch.arange(m0, m0 + len(x), device="cuda") + n - m
                sc = torch.where(torch.arange(n, device="cuda") <= at[:, None, None], sc, -math.inf)
                o[m0:m0 + 256, h * R:(h + 1) * R] = torch.softmax(sc, -1) @ v
        out.append(o)
    return torch.cat(out)


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    H, D = case["kv_heads"], case["dim"]
    if case["kind"] in ("store", "read"):
        n = case["tokens"] * H * 2 * D
        held = case["tokens"] * (H * (2 * D + 2))
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": float(n * size * (case["kind"] == "store") + held + 2 * n + 4 * case["tokens"]), "flops": 0.0}
    lengths, new = _lengths(case)
    seen = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lengths, new)) if case["kind"] == "chunk" else sum(lengths)
    return {"bytes": float(sum(lengths) * H * (2 * D + 2) + 4 * sum(new) * case["heads"] * D), "flops": 4.0 * seen * case["heads"] * D}
