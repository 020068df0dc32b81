"""Distillation from a teacher's most likely tokens, through the lm head and without a ``[N, V]`` logits tensor.

``lm_head_distill(hidden, weight, labels, teacher_ids, teacher_logprobs, teacher_rest)`` compares, per row, the student's distribution
``softmax(hidden @ weight^T * inv_temperature)`` with a teacher's, of which the log-probabilities of ``K`` tokens are known and, with
``teacher_rest``, the log of the mass of all others, which then are one class more (:func:`~.logprob.top_logprobs` gives the three).  Over
these classes, q the teacher's masses and p the student's, the divergence is ``(1 - reverse) KL(q, p) + reverse KL(p, q)``; without
``teacher_rest`` both sums run over the named tokens alone (p stays normalised over the whole vocabulary).

On CUDA the vocabulary product runs on tcgen05 CTA pairs with an epilogue that reduces every 128 columns to records without the named
tokens, whose logits are dot products of their own (``csrc/distill.cu``); the backward pass forms d(logits) in bf16 a chunk of rows at a time, from the
exponentials that the forward pass kept or from the logits once more, and feeds two products.  CPU tensors use the
fp32 expression below (the oracle of the GPU tests).
"""
from __future__ import annotations

import ctypes
import functools
from typing import Dict, Optional, Tuple

import torch

from . import _lib
from .logprob import _BWD_BUDGET, _BWD_ROWS, _bwd_rows
from ..utils import memory_budget

MOST_NAMED = 256        # tokens that a row may name

_FN: Dict[str, object] = {}


def _fn(name: str):
    if not _FN:
        c, fns = ctypes, {}
        vp, i, ll, f = c.c_void_p, c.c_int, c.c_longlong, c.c_float
        fns["fwd"] = _lib.declare("apb_lmhead_distill_fwd", [vp] * 18 + [i, i, i, i, ll, ll, f, f, vp])
        fns["bwd"] = _lib.declare("apb_lmhead_distill_bwd", [vp] * 21 + [i, i, i, i, i, ll, ll, f, vp])
        _FN.update(fns)              # in one step: another thread may be looking
    return _FN[name]


def first_entries(ids: torch.Tensor, vocab: int) -> torch.Tensor:
    """Which entries of ``ids [N, K]`` count: those that name a token of the vocabulary, of a token named again the first one."""
    there = (ids >= 0) & (ids < vocab)
    again = (ids[:, :, None] == ids[:, None, :]).tril(-1).any(-1)
    return there & ~again


def _times(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """``x y``; 0, also in its gradients, where ``x`` is: a class without mass adds nothing, whatever its logarithm is."""
    return torch.where(x > 0, x * torch.where(x > 0, y, 0.0), 0.0)


def distill_ref(hidden, weight, labels, teacher_ids, teacher_logprobs, teacher_rest=None, inv_temperature=1.0, reverse: float = 0.0,
                with_entropy: bool = True, dtype: torch.dtype = torch.float32):
    """Differentiable expression of :func:`lm_head_distill` in ``dtype``."""
    V = weight.shape[0]
    it = inv_temperature.to(dtype)[:, None] if torch.is_tensor(inv_temperature) else float(inv_temperature)
    z = (hidden.to(dtype) @ weight.to(dtype).t()) * it
    log_p = torch.log_softmax(z, -1)
    counts = first_entries(teacher_ids, V)
    ids = torch.where(counts, teacher_ids, 0).long()
    lq = torch.where(counts, teacher_logprobs.detach().to(dtype), 0.0)
    q = torch.where(counts, lq.exp(), 0.0)
    lp = torch.where(counts, log_p.gather(1, ids), 0.0)
    p = torch.where(counts, lp.exp(), 0.0)
    value = (1 - reverse) * _times(q, lq - lp).sum(-1)
    if reverse:
        value = value + reverse * _times(p, lp - lq).sum(-1)
    if teacher_rest is not None:
        lqr = teacher_rest.detach().to(dtype)
        named = torch.zeros(z.shape, dtype=torch.bool, device=z.device)
        rows = torch.arange(z.shape[0], device=z.device)[:, None].expand_as(ids)
        named[rows[counts], ids[counts]] = True
        left = ~named.all(-1)
        lpr = torch.logsumexp(torch.where(named & left[:, None], float("-inf"), log_p), -1)
        value = value + (1 - reverse) * _times(lqr.exp(), lqr - torch.where(left, lpr, float("-inf")))
        if reverse:
            value = value + reverse * _times(torch.where(left, lpr.exp(), 0.0), lpr - lqr)
    lab = labels.long()
    logprob = log_p.gather(1, lab[:, None]).squeeze(-1)
    entropy = -(log_p.exp() * log_p).sum(-1) if with_entropy else None
    return value, logprob, entropy


def _split_pays(n: int, H: int, pairs: int) -> bool:
    """Whether a product ``[n, H]`` over the vocabulary is cut into parts of it that add up in fp32: where its tiles of 256 x 256 leave much of
    their last wave of CTA pairs idle (4096 x 2560: 160 tiles, 2.2 waves, 2.6 ms; in six parts 2.1 ms)."""
    tiles = -(-n // 256) * -(-H // 256)
    return tiles < 0.85 * pairs * -(-tiles // pairs)


# Probabilities from which on keeping them pays.  With the memory at hand it saves 20 us of 360 at 1e7 of them, 56 of 703 to 222 of 2186 at 6e7
# (H = 1024 and 2560), and costs 22 of 205 at 1e6; but where the allocator has not enough, asking the driver takes 150 us to 2 ms.
_KEEP_FROM = 1 << 26


def _keep_pays(N: int, V: int, device) -> bool:
    """Whether the forward pass keeps the exponentials of its logits in bf16 for the backward pass, which then need not form the logits again
    (a quarter of its products): where the device has room for them and for the gradient beside.  Kept ones are rounded to bf16 once more, so that
    the last bits of a gradient depend on it."""
    size = 2 * N * V
    return N * V >= _KEEP_FROM and size <= _BWD_BUDGET // 2 and memory_budget.spare_bytes(device, 3 * size) >= 3 * size


@functools.lru_cache(maxsize=None)
def _pairs(device) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count // 2


def _row_places(rows: torch.Tensor, N: int, K: int) -> Tuple[int, int, int, int, int]:
    """Addresses of logits ``[N, K + 1]`` and log-sum-exp ``[N]`` (fp64), the others' references and coefficients ``[N]`` and the named
    gradients ``[N, K]`` in the block that a forward pass keeps."""
    logit = rows.data_ptr()
    lse = logit + 8 * N * (K + 1)
    return logit, lse, lse + 8 * N, lse + 12 * N, lse + 16 * N


class _LmHeadDistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ids, teacher, rest, inv_temp_t, inv_temp_s, reverse, with_entropy, bwd_chunk, grads):
        N, H = hidden.shape
        V, K = weight.shape[0], ids.shape[1]
        dev, f32 = hidden.device, torch.float32
        tiles = (V + 127) // 128
        partial = torch.empty((N, tiles, 4), device=dev, dtype=f32)
        in_order = torch.empty(N * K + (N * tiles + 1) // 2, device=dev, dtype=torch.int32)
        value, lp, ent = (torch.empty(N, device=dev, dtype=f32) for _ in range(3))
        # what the backward pass takes up again: logits [N, K + 1] of the named tokens and the label and log-sum-exp [N] in 64 bits, reference and
        # coefficient of the others of every row, gradients [N, K] of the named ones (one block: an allocation costs the host 3 us) and the
        # others' exponentials
        rows = torch.empty(N * (3 * K + 6), device=dev, dtype=f32)
        logit, lse, ref, others, named = _row_places(rows, N, K)
        # not by what memory happens to be free where the caller bounds it, or wants the same bits each time
        may = bwd_chunk is None and not torch.are_deterministic_algorithms_enabled()
        keep = grads and may and any(ctx.needs_input_grad[:2]) and _keep_pays(N, V, dev)
        kept = torch.empty((N, V), device=dev, dtype=torch.bfloat16) if keep else None
        opt = lambda t: None if t is None else t.data_ptr()                                  # noqa: E731
        _lib.check(_fn("fwd")(hidden.data_ptr(), weight.data_ptr(), labels.data_ptr(), ids.data_ptr(), teacher.data_ptr(), opt(rest),
                              opt(inv_temp_t), partial.data_ptr(), in_order.data_ptr(), logit, value.data_ptr(), lp.data_ptr(),
                              ent.data_ptr(), lse, ref, others, named, opt(kept), N, V, H, K, hidden.stride(0), weight.stride(0),
                              inv_temp_s, reverse, _lib.stream_ptr()), "apb_lmhead_distill_fwd")
        ctx.save_for_backward(hidden, weight, labels, ids, inv_temp_t, rows, ent, kept, None if kept is None else partial)
        ctx.inv_temp_s, ctx.with_entropy, ctx.bwd_chunk = inv_temp_s, with_entropy, bwd_chunk
        ctx.set_materialize_grads(False)
        return value, lp, (ent if with_entropy else None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_value, g_lp, g_ent):
        hidden, weight, labels, ids, it, rows, ent, kept, partial = ctx.saved_tensors
        N, H = hidden.shape
        V, K = weight.shape[0], ids.shape[1]
        dev = hidden.device
        want_h, want_w = ctx.needs_input_grad[:2]
        whole = lambda g: g if g is None or g.dtype is torch.float32 and g.is_contiguous() else g.to(torch.float32).contiguous()  # noqa: E731
        g_value, g_lp, g_ent = whole(g_value), whole(g_lp), whole(g_ent) if ctx.with_entropy else None
        at = lambda t, s, size: None if t is None else t.data_ptr() + s * size               # noqa: E731
        chunk = ctx.bwd_chunk
        if chunk is None:
            fixed = N <= _BWD_ROWS or torch.are_deterministic_algorithms_enabled()
            chunk = _bwd_rows(N, V, 0 if fixed else memory_budget.spare_bytes(dev, _BWD_BUDGET))
        buf_rows = min(chunk, N) if ctx.bwd_chunk or N <= _BWD_ROWS else -(-chunk // _BWD_ROWS) * _BWD_ROWS
        buf = torch.empty((buf_rows, V), device=dev, dtype=torch.bfloat16)
        scratch = torch.empty(3 * min(chunk, N), device=dev, dtype=torch.float32)
        d_hidden = torch.empty((N, H), device=dev, dtype=hidden.dtype) if want_h else None
        acc = getattr(weight, "grad_f32", None) if want_w else None
        # one chunk: the weight's gradient leaves its product in its own type; several add up in fp32
        dw = None if not want_w or acc is not None else torch.empty((V, H), device=dev, dtype=weight.dtype) if chunk >= N else \
            torch.zeros((V, H), device=dev, dtype=torch.float32)
        pairs = _pairs(dev)
        total = torch.empty((min(chunk, N), H), device=dev, dtype=torch.float32) if want_h and _split_pays(min(chunk, N), H, pairs) else None
        into = acc if acc is not None else dw
        logit, lse, ref, others, named = _row_places(rows, N, K)
        tiles = (V + 127) // 128
        for s in range(0, N, chunk):
            n = min(chunk, N - s)
            _lib.check(_fn("bwd")(at(hidden, s, 2 * hidden.stride(0)), weight.data_ptr(), at(ids, s, 4 * K), at(labels, s, 4), at(it, s, 4),
                                  logit + 8 * s * (K + 1), named + 4 * s * K, others + 4 * s, lse + 8 * s, ref + 4 * s,
                                  at(ent, s, 4), at(g_value, s, 4), at(g_lp, s, 4), at(g_ent, s, 4), at(kept, s, 2 * V), at(partial, s, 16 * tiles),
                                  scratch.data_ptr(), buf.data_ptr(), at(d_hidden, s, 2 * H), at(total, 0, 4), at(into, 0, 4),
                                  into is not None and into.dtype == torch.float32, n, V, H, K, hidden.stride(0), weight.stride(0),
                                  ctx.inv_temp_s, _lib.stream_ptr()), "apb_lmhead_distill_bwd")
        if dw is not None and dw.dtype != weight.dtype:
            dw = dw.to(weight.dtype)
        return (d_hidden, dw) + (None,) * 10


def lm_head_distill(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, teacher_ids: torch.Tensor,
                    teacher_logprobs: torch.Tensor, teacher_rest: Optional[torch.Tensor] = None, inv_temperature=1.0,
                    reverse: float = 0.0, with_entropy: bool = True, bwd_chunk: Optional[int] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """``hidden [N, H]``, ``weight [V, H]``, ``labels [N]``, ``teacher_ids [N, K]`` (integers), ``teacher_logprobs [N, K]``,
    ``teacher_rest [N]`` or None -> ``(divergence [N], logprob [N], entropy [N] or None)``, fp32, all three differentiable in ``hidden`` and
    ``weight`` (the teacher's numbers get no gradient).  ``logprob`` and ``entropy`` are those of :func:`~.logprob.lm_head_logprobs`.

    An entry of ``teacher_ids`` outside the vocabulary (-1 by custom) names nothing; a token named again in a row counts once, by its
    first entry.  A row that names nothing has divergence 0 without ``teacher_rest``.  A class that the teacher gives no mass (a
    log-probability of ``-inf``) makes the reverse divergence infinite.  ``inv_temperature`` is a float or a per-row tensor ``[N]``.
    On CUDA: bf16 hidden states and weights, H and V multiples of 8, K at most 256.

    ``bwd_chunk``: rows of d(logits) that the backward pass forms at a time.  Without it the backward pass takes more memory where the device has
    it to spare: the probabilities of the forward pass, rounded to bf16 (2 N V bytes, from 2^26 of them on), and more rows at a time.  With it, or under
    ``torch.use_deterministic_algorithms``, what is computed does not depend on that.  d(logits) is a bf16 tensor either way, so that a gradient
    is off by 2.3 to 2.5e-3 of its norm, 1.7e-3 of it its own rounding."""
    if hidden.dim() != 2 or weight.dim() != 2 or hidden.shape[1] != weight.shape[1]:
        raise ValueError(f"hidden {list(hidden.shape)} and weight {list(weight.shape)} must be [N, H] and [V, H]")
    N, H = hidden.shape
    V = weight.shape[0]
    if teacher_ids.dim() != 2 or teacher_ids.shape[0] != N or teacher_logprobs.shape != teacher_ids.shape:
        raise ValueError(f"teacher_ids {list(teacher_ids.shape)} and teacher_logprobs {list(teacher_logprobs.shape)} must be [{N}, K] both")
    if teacher_ids.dtype not in (torch.int32, torch.int64) or not teacher_logprobs.is_floating_point():
        raise ValueError(f"teacher_ids must be int32 or int64, teacher_logprobs floating: {teacher_ids.dtype}, {teacher_logprobs.dtype}")
    for name, t in (("labels", labels), ("teacher_rest", teacher_rest), ("inv_temperature", inv_temperature)):
        if torch.is_tensor(t) and t.shape != (N,):
            raise ValueError(f"{name} must be [{N}], got {list(t.shape)}")
    if not 0.0 <= float(reverse) <= 1.0:
        raise ValueError(f"reverse must lie between 0 (teacher to student) and 1 (student to teacher), got {reverse}")
    tensors = {"weight": weight, "labels": labels, "teacher_ids": teacher_ids, "teacher_logprobs": teacher_logprobs,
               "teacher_rest": teacher_rest, "inv_temperature": inv_temperature}
    for name, t in tensors.items():
        if torch.is_tensor(t) and t.device != hidden.device:
            raise ValueError(f"{name} lives on {t.device}, hidden on {hidden.device}")
    if not hidden.is_cuda:
        return distill_ref(hidden, weight, labels, teacher_ids, teacher_logprobs, teacher_rest, inv_temperature, float(reverse), with_entropy)
    if hidden.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise ValueError(f"hidden and weight must be bf16 on a GPU, got {hidden.dtype} and {weight.dtype}")
    if H % 8 or V % 8 or V == 0 or H == 0 or teacher_ids.shape[1] > MOST_NAMED:
        raise ValueError(f"H = {H} and V = {V} must be multiples of 8, K = {teacher_ids.shape[1]} at most {MOST_NAMED}")
    if N == 0:
        # connected to its inputs, so that a shard without rows still has a gradient of zeros
        z = (hidden.sum() + weight[:0].sum()) * 0.0 + hidden.new_zeros(0, dtype=torch.float32)
        return z, z, (z if with_entropy else None)
    if hidden.get_device() != torch._C._cuda_getDevice():
        with torch.cuda.device(hidden.device):
            return lm_head_distill(hidden, weight, labels, teacher_ids, teacher_logprobs, teacher_rest, inv_temperature, reverse, with_entropy,
                                   bwd_chunk)
    if weight.stride(1) != 1 or weight.stride(0) % 8 or weight.stride(0) < H or weight.data_ptr() % 16:
        raise ValueError("weight must have whole rows on 16-byte boundaries")
    # expanded rows too; contiguous() would leave dense rows off their boundary, and a single row of any stride, as they are
    if hidden.stride(1) != 1 or hidden.stride(0) % 8 or hidden.stride(0) < H or hidden.data_ptr() % 16:
        hidden = hidden.clone(memory_format=torch.contiguous_format)
    whole = lambda t, dtype: t if t.dtype is dtype and t.is_contiguous() and not t.requires_grad else t.detach().to(dtype).contiguous()  # noqa: E731
    if teacher_ids.dtype == torch.int64:         # before 32 bits cut them
        teacher_ids = torch.where((teacher_ids < 0) | (teacher_ids >= V), -1, teacher_ids)
    it_t = whole(inv_temperature, torch.float32) if torch.is_tensor(inv_temperature) else None
    return _LmHeadDistillFn.apply(
        hidden, weight, whole(labels, torch.int32), whole(teacher_ids, torch.int32), whole(teacher_logprobs, torch.float32),
        None if teacher_rest is None else whole(teacher_rest, torch.float32), it_t, 1.0 if it_t is not None else float(inv_temperature),
        float(reverse), with_entropy, bwd_chunk, torch.is_grad_enabled())      # which is off within the function, whatever its inputs need
