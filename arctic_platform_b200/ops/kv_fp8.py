"""Paged key/value cache in 8 bits: rows quantised as they are written and read back, attention over it.

A page of 16 tokens is a block of bytes per key head: 16 rows of ``D`` key codes (e4m3), 16 rows of value codes, 32 exponents.  A
row of a token stands for ``code * 2^(byte - 127)``, the exponent being the least one, of -100 to 119, with which the row's largest
magnitude is at most 448: half the bytes of bf16 and a 128th of those for ``D`` = 128, every value exactly a bf16 number and off by at most
2^-4 of itself (2^-10 of 2^exponent where it is smaller than 2^-6 of that).  A row's codes depend on that row alone: neither the
order nor the portions in which a page is filled change what it holds.

* :func:`write` quantises rows into their slots, :func:`read` gives them back; :func:`norm_rope_write` does it behind the projection of a
  decode step;
* :func:`decode_attention` is the attention of one query token per sequence (page tables and lengths on the device, as in a captured
  decode step), :func:`chunk_attention` that of the last tokens of each sequence, causal, by a plan that is made once per step.  Scores are
  fp32 numbers: a query's largest magnitude times that of a key has to be below 2e38.

CUDA tensors run ``kv_fp8_*.cu``; CPU tensors run the plain PyTorch expressions below (the oracle of the GPU tests).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from ..utils import checked
from ..utils.transfer_stats import to_device

PAGE = 16
LEAST_EXPONENT, MOST_EXPONENT = -100, 119
DIMS = (64, 128)

_FN: Dict[str, object] = {}


def _fn(name: str):
    if not _FN:
        c, fns = ctypes, {}
        vp, i, ll, f = c.c_void_p, c.c_int, c.c_longlong, c.c_float
        fns["write"] = _lib.declare("apb_kv8_write", [vp, ll, ll, vp, ll, ll, vp, vp, i, i, i, i, i, vp])
        fns["read"] = _lib.declare("apb_kv8_read", [vp, vp, vp, vp, i, i, i, i, i, vp])
        fns["qkv"] = _lib.declare("apb_kv8_qkv_post", [vp, ll] + [vp] * 8 + [i, i, i, i, i, i, f, vp])
        fns["decode"] = _lib.declare("apb_kv8_decode", [vp, ll, vp, vp, ll, i, i, vp, vp, vp, ll, i, i, i, i, i, f, vp, vp])
        fns["scratch"] = _lib.declare("apb_kv8_decode_scratch", [i, i, i, i, i], ll)
        fns["few"] = _lib.declare("apb_kv8_few", [vp, ll, vp, vp, ll, i, i, vp, vp, vp, ll, i, i, i, i, i, i, f, vp])
        fns["chunk"] = _lib.declare("apb_kv8_chunk", [vp, ll, vp, vp, ll, vp, vp, i, vp, i, i, i, vp, vp, ll, i, i, i, i, f, vp])
        _FN.update(fns)              # in one step: another thread may be looking
    return _FN[name]


def block_bytes(head_dim: int) -> int:
    """Bytes of the 16 tokens of a page and key head."""
    return 2 * PAGE * head_dim + 2 * PAGE


class Fp8KVCache:
    """``data [..., pages, key heads, block]`` uint8: the blocks of one layer, or of all layers in front (:meth:`layer`)."""

    __slots__ = ("data", "head_dim", "num_pages", "num_kv_heads", "one_layer", "index")

    def __init__(self, data: torch.Tensor, head_dim: int):
        if head_dim not in DIMS:
            raise ValueError(f"head_dim {head_dim}: the 8-bit cache holds heads of {DIMS[0]} or {DIMS[1]}")
        if data.dtype != torch.uint8 or data.dim() not in (3, 4) or data.shape[-1] != block_bytes(head_dim):
            raise ValueError(f"data must be uint8 [(layers,) pages, heads, {block_bytes(head_dim)}], got {data.dtype} {tuple(data.shape)}")
        if min(data.shape[:-1]) < 1:
            raise ValueError("a cache has at least one page and head")
        if not data.is_contiguous() or data.data_ptr() % 16:
            raise ValueError("data must be contiguous and begin on a 16-byte boundary")
        self.data, self.head_dim = data, head_dim
        # plain numbers: a decode step asks for them in every layer
        self.num_pages, self.num_kv_heads, self.one_layer, self.index = data.shape[-3], data.shape[-2], data.dim() == 3, data.get_device()

    @staticmethod
    def zeros(num_pages: int, num_kv_heads: int, head_dim: int, device="cuda", layers: Optional[int] = None) -> "Fp8KVCache":
        shape = (num_pages, num_kv_heads, block_bytes(head_dim))
        return Fp8KVCache(torch.zeros(shape if layers is None else (layers,) + shape, device=device, dtype=torch.uint8), head_dim)

    def layer(self, i: int) -> "Fp8KVCache":
        return Fp8KVCache(self.data[i], self.head_dim)

    def nbytes(self) -> int:
        return self.data.numel()

    def parts(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Views: key codes and value codes ``[..., 16, D]``, exponent bytes ``[..., 8, 2, 2]`` (token % 8; key or value; token // 8)."""
        n = PAGE * self.head_dim
        k, v = (self.data[..., i * n:(i + 1) * n].unflatten(-1, (PAGE, self.head_dim)) for i in (0, 1))
        return k, v, self.data[..., 2 * n:].unflatten(-1, (8, 2, 2))


def _refuse(cache: Fp8KVCache, **tensors) -> None:
    """Says what is wrong with where the tensors are."""
    if not cache.one_layer:
        raise ValueError("a cache of several layers: take one with .layer(i)")
    for name, t in tensors.items():
        if t.get_device() != cache.index:
            raise ValueError(f"{name} lives on {t.device}, not on {cache.data.device}")


def _elsewhere(cache: Fp8KVCache) -> bool:
    """The cache is on another GPU than the current one."""
    return cache.index != torch._C._cuda_getDevice()


# --------------------------------------------------------------------------------------------- rows
def quantise_ref(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows ``[..., D]`` to codes (uint8) and exponent bytes ``[...]``."""
    x = x.float()
    most = torch.nan_to_num(x.abs(), nan=0.0).amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(most)                       # 448 = 0.875 * 2^9
    e = torch.where(most > 0, exponent - 9 + (mantissa > 0.875), LEAST_EXPONENT)
    e = torch.where(torch.isinf(most), MOST_EXPONENT, e).clamp(LEAST_EXPONENT, MOST_EXPONENT)
    codes = (x * torch.exp2(-e.float())).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), (e + 127).squeeze(-1).to(torch.uint8)


def values_ref(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """Codes ``[..., D]`` and exponent bytes ``[...]`` to fp32."""
    return codes.contiguous().view(torch.float8_e4m3fn).float() * torch.exp2(byte.float() - 127)[..., None]


def _check_slots(cache: Fp8KVCache, slots: torch.Tensor, distinct: bool) -> None:
    if slots.dtype is not torch.int32 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError(f"slots must be int32 [rows] with neighbouring elements, got {slots.dtype} {list(slots.shape)}")
    if not cache.one_layer or slots.get_device() != cache.index:
        _refuse(cache, slots=slots)
    if checked.enabled() and checked.active_for(slots):
        checked.check_range("slots", slots, -(1 << 31), cache.num_pages * PAGE)
        if distinct:
            checked.check_distinct("slots", slots)


def write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, cache: Fp8KVCache) -> None:
    """``k``, ``v [T, heads, D]`` (bf16 or fp32; tokens and heads may be strided, as the columns of a projection are) into
    ``slots [T]`` int32 = page * 16 + token in the page; rows of slots below 0 are left out.  A slot is named once in a call.

    Magnitudes above 448 * 2^119 (2.98e38), infinities among them, become that; what is not a number stays none and leaves the
    rest of its row alone."""
    _check_slots(cache, slots, True)
    data, shape, dt = cache.data, (slots.shape[0], cache.num_kv_heads, cache.head_dim), k.dtype
    index = cache.index
    if (v.dtype is not dt or (dt is not torch.bfloat16 and dt is not torch.float32) or k.shape != shape or v.shape != shape
            or k.get_device() != index or v.get_device() != index):
        for name, t in (("k", k), ("v", v)):
            if t.dtype is not dt or t.shape != shape or (dt is not torch.bfloat16 and dt is not torch.float32):
                raise ValueError(f"{name} must be bf16 or fp32 {list(shape)}, got {t.dtype} {list(t.shape)}")
        _refuse(cache, k=k, v=v)
    T, H, D = shape
    if T == 0:
        return
    if index < 0:
        ck, cv, ex = cache.parts()
        at = slots[slots >= 0].long()
        if at.numel() and int(at.max()) >= cache.num_pages * PAGE:
            raise ValueError("slots: beyond the cache's pages")
        page, t = at // PAGE, at % PAGE
        for w, (codes, x) in enumerate(((ck, k), (cv, v))):
            c, e = quantise_ref(x[slots >= 0])
            codes[page, :, t] = c
            ex[page, :, t % 8, w, t // 8] = e
        return
    if _elsewhere(cache):
        with torch.cuda.device(cache.index):
            return write(k, v, slots, cache)
    k, k0, k1 = _rows_aligned(k)
    v, v0, v1 = _rows_aligned(v)
    _lib.check(_fn("write")(k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, slots.data_ptr(), data.data_ptr(), T, H, D, cache.num_pages,
                            dt is torch.float32, _lib.stream_ptr()), "kv8_write")


def _rows_aligned(t: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """``t [T, heads, D]`` itself where its rows are whole and begin on 16-byte boundaries, else a copy; its strides."""
    a, b, c = t.stride()
    if c != 1 or (a | b) % (16 // t.element_size()) or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        a, b, _ = t.stride()
    return t, a, b


def _rows(T: int, H: int, D: int, like: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """New rows ``[T, H, D]`` on the device of ``like`` (with the strides named: 0.8 us of host time less than ``torch.empty``)."""
    return torch.empty_strided((T, H, D), (H * D, D, 1), device=like.device, dtype=dtype)


def read(cache: Fp8KVCache, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that ``slots [T]`` hold, ``[T, heads, D]`` each, exact in ``dtype`` (bf16 or fp32); zeros for slots below 0."""
    _check_slots(cache, slots, False)
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise ValueError(f"rows are read as bf16 or fp32, not {dtype}")
    data, T, H, D = cache.data, slots.shape[0], cache.num_kv_heads, cache.head_dim
    if cache.index < 0:
        if T and int(slots.max()) >= cache.num_pages * PAGE:
            raise ValueError("slots: beyond the cache's pages")
        ck, cv, ex = cache.parts()
        at = slots.long().clamp_min(0)
        page, t, keep = at // PAGE, at % PAGE, (slots >= 0)[:, None, None]
        return tuple(torch.where(keep, values_ref(c[page, :, t], ex[page, :, t % 8, w, t // 8]), 0.0).to(dtype) for w, c in enumerate((ck, cv)))
    if _elsewhere(cache):
        with torch.cuda.device(cache.index):
            return read(cache, slots, dtype)
    k, v = _rows(T, H, D, data, dtype), _rows(T, H, D, data, dtype)
    if T:
        _lib.check(_fn("read")(data.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), T, H, D, cache.num_pages,
                               dtype is torch.float32, _lib.stream_ptr()), "kv8_read")
    return k, v


def norm_rope_write(acc: torch.Tensor, q_norm: Optional[torch.Tensor], k_norm: Optional[torch.Tensor], rope: Tuple[torch.Tensor, torch.Tensor],
                    positions: torch.Tensor, slots: torch.Tensor, cache: Fp8KVCache, heads: int, eps: float) -> torch.Tensor:
    """A decode step behind its qkv projection (CUDA only): ``acc [B, (heads + 2 * key heads) * D]`` fp32 sums, left as zeros for the next
    ones to be added to; RMSNorm per head (weights ``[D]`` bf16, or None) and rotate-half RoPE (``cos, sin [positions, D / 2]`` fp32) of
    q and k at ``positions [B]`` int32.  Returns q ``[B, heads, D]`` bf16; k and v are rounded to bf16 and written as :func:`write` does.
    A position that the tables do not have gives zeros for q, and k and v are not written; it is reported (:func:`_lib.check_status`) where the
    row has a slot."""
    _check_slots(cache, slots, True)
    data, B, H, D = cache.data, slots.shape[0], cache.num_kv_heads, cache.head_dim
    width = (heads + 2 * H) * D
    if heads < 1 or acc.dtype is not torch.float32 or acc.shape != (B, width) or acc.stride(1) != 1 or (B > 1 and acc.stride(0) < width):
        raise ValueError(f"acc must be fp32 {[B, width]} with whole rows of their own, got {acc.dtype} {list(acc.shape)}")
    if positions.dtype is not torch.int32 or positions.shape != slots.shape or not positions.is_contiguous():
        raise ValueError("positions must be int32, one per row")
    cos, sin = rope
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype is not torch.float32 or t.dim() != 2 or t.shape != (cos.shape[0], D // 2) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous fp32 [positions, {D // 2}], as many as the other one, got {t.dtype} {list(t.shape)}")
    norms = {name: t for name, t in (("q_norm", q_norm), ("k_norm", k_norm)) if t is not None}
    for name, t in norms.items():
        if t.dtype is not torch.bfloat16 or t.shape != (D,) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous bf16 [{D}], got {t.dtype} {list(t.shape)}")
    _refuse(cache, acc=acc, positions=positions, cos=cos, sin=sin, **norms)
    if cache.index < 0:
        raise ValueError("norm_rope_write runs on a GPU")
    if checked.enabled() and checked.active_for(positions):
        checked.check_range("positions", positions, 0, cos.shape[0], where=slots >= 0)
    if _elsewhere(cache):
        with torch.cuda.device(cache.index):
            return norm_rope_write(acc, q_norm, k_norm, rope, positions, slots, cache, heads, eps)
    q = torch.empty((B, heads, D), device=data.device, dtype=torch.bfloat16)
    _lib.check(_fn("qkv")(acc.data_ptr(), acc.stride(0), _lib.ptr(q_norm), _lib.ptr(k_norm), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(),
                          slots.data_ptr(), q.data_ptr(), data.data_ptr(), B, heads, H, D, cache.num_pages, cos.shape[0], float(eps),
                          _lib.stream_ptr()), "kv8_qkv_post")
    return q


# --------------------------------------------------------------------------------------------- attention
def _check_queries(q: torch.Tensor, cache: Fp8KVCache, out: Optional[torch.Tensor]) -> Tuple[torch.Tensor, int]:
    """The queries, copied where their rows are not whole, off the 16-byte boundaries or one over another (a tensor map wants strides that
    grow); the distance of their rows."""
    rows, heads, dim = q.shape if q.dim() == 3 else (0, 0, 0)
    if q.dtype is not torch.bfloat16 or dim != cache.head_dim or heads == 0 or heads % cache.num_kv_heads:
        raise ValueError(f"q must be bf16 [rows, a multiple of {cache.num_kv_heads} heads, {cache.head_dim}], got {q.dtype} {list(q.shape)}")
    if not cache.one_layer or q.get_device() != cache.index:
        _refuse(cache, q=q)
    a, b, c = q.stride()
    if out is not None:
        if (out.dtype is not torch.bfloat16 or out.shape != q.shape or out.stride(2) != 1 or out.stride(1) != dim
                or (rows > 1 and out.stride(0) < heads * dim)):
            raise ValueError("out must be bf16 of q's shape with whole rows of their own")
        if out.get_device() != cache.index:
            _refuse(cache, out=out)
    if c != 1 or b != dim or a % 8 or a < heads * dim or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        a = heads * dim
    return q, a


def context_ref(cache: Fp8KVCache, pages: torch.Tensor, n: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of the first ``n`` tokens on ``pages``, ``[n, heads, D]`` fp32."""
    t = torch.arange(n, device=pages.device)
    return read(cache, (pages.long()[t // PAGE] * PAGE + t % PAGE).to(torch.int32), torch.float32)


def attention_ref(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, last: torch.Tensor, scale: float) -> torch.Tensor:
    """``q [rows, Hq, D]`` over ``k``, ``v [n, Hkv, D]`` up to token ``last [rows]``; zeros where a row sees nothing."""
    rep = q.shape[1] // k.shape[1]
    s = torch.einsum("ihd,thd->hit", q.to(k.dtype), k.repeat_interleave(rep, 1)) * scale
    seen = torch.arange(k.shape[0], device=q.device) <= last[:, None]
    s = s.masked_fill(~seen, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).nan_to_num(neginf=0.0)) if k.shape[0] else s
    total = p.sum(-1)
    o = torch.einsum("hit,thd->ihd", p, v.repeat_interleave(rep, 1))
    return o / torch.where(total == 0, 1.0, total).t()[..., None]


def _refuse_tables(cache: Fp8KVCache, page_table: torch.Tensor, lengths: torch.Tensor, B: int, what: str = "lengths") -> None:
    """Says what is wrong with a batch's tables."""
    for name, t, dims in (("page_table", page_table, 2), (what, lengths, 1)):
        if t.dtype is not torch.int32 or t.dim() != dims or t.shape[0] != B or (t.stride(dims - 1) != 1 and t.numel()):
            shape = f"[{B}, pages]" if dims == 2 else [B]
            raise ValueError(f"{name} must be int32 {shape} with neighbouring elements, got {t.dtype} {list(t.shape)}")
        if t.get_device() != cache.index:
            _refuse(cache, **{name: t})


def decode_attention(q: torch.Tensor, cache: Fp8KVCache, page_table: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None, longest: Optional[int] = None, active: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``q [B, Hq, D]`` bf16, one token per sequence, over the first ``lengths [B]`` (int32) tokens on the pages ``page_table
    [B, max_pages]`` (int32) -> ``[B, Hq, D]`` bf16; zeros for sequences of length 0.  Query head ``h`` reads key head
    ``h // (Hq // Hkv)``; ``scale``: of the scores, ``D ** -0.5`` if None.  Entries of the table behind a sequence's pages are not looked at.

    ``longest``: about how long the longest sequence is or will be, where the table is much wider than that; the kernel is chosen by it,
    the result does not depend on it but for last bits.  ``active [B]`` int32: sequences where it is not above 0 are taken as empty, whatever
    their length says."""
    q, ldq = _check_queries(q, cache, out)
    B, Hq, D = q.shape
    index = cache.index
    if (page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[0] != B
            or (page_table.stride(1) != 1 and page_table.numel())
            or lengths.dtype is not torch.int32 or lengths.shape != (B,) or (lengths.stride(0) != 1 and B)
            or page_table.get_device() != index or lengths.get_device() != index):
        _refuse_tables(cache, page_table, lengths, B)
    if active is not None and (active.dtype is not torch.int32 or active.shape != (B,) or (active.stride(0) != 1 and B)
                               or active.get_device() != index):
        _refuse_tables(cache, page_table, active, B, "active")
    data, scale = cache.data, D ** -0.5 if scale is None else float(scale)
    if checked.enabled() and checked.active_for(q):
        checked.check_page_table("page_table", page_table, lengths if active is None else lengths * (active > 0), cache.num_pages, PAGE)
    if out is None:
        out = _rows(B, Hq, D, data, torch.bfloat16)
    if B == 0:
        return out
    if index < 0:
        for b, n in enumerate((lengths if active is None else lengths * (active > 0)).tolist()):
            k, v = context_ref(cache, page_table[b], n)
            out[b:b + 1] = attention_ref(q[b:b + 1].float(), k, v, torch.tensor([n - 1]), scale).to(q.dtype)
        return out
    if _elsewhere(cache):
        with torch.cuda.device(cache.index):
            return decode_attention(q, cache, page_table, lengths, scale, out, longest, active)
    if out.stride(0) % 8 or out.data_ptr() % 16:             # rows off the 16-byte boundaries: by way of a copy
        return out.copy_(decode_attention(q, cache, page_table, lengths, scale, None, longest, active))
    wide = page_table.shape[1]
    pages = wide if longest is None else min(wide, (longest + PAGE - 1) // PAGE)
    need = _fn("scratch")(B, pages, Hq, cache.num_kv_heads, D)
    scratch = torch.empty(need, device=data.device, dtype=torch.uint8) if need else None          # kept until the launch has been made
    _lib.check(_fn("decode")(q.data_ptr(), ldq, data.data_ptr(), page_table.data_ptr(), page_table.stride(0), wide, cache.num_pages,
                             lengths.data_ptr(), _lib.ptr(active), out.data_ptr(), out.stride(0), B, pages, Hq, cache.num_kv_heads, D, scale,
                             _lib.ptr(scratch), _lib.stream_ptr()), "kv8_decode")
    return out


@dataclass
class _Work:
    """What the CTAs of chunk attention do (``csrc/runtime_kv8.cpp``): items, where each CTA's begin, joins of items cut along the keys."""
    items: np.ndarray
    first: np.ndarray
    joins: np.ndarray
    part_tiles: int           # tiles of 128 rows of scratch
    ctas: int                 # or pairs of them
    form: int                 # how items are taken: one or two tiles, one, one or two of 256 rows by two CTAs

    @property
    def one_tile(self) -> bool:
        return self.form == 1


def _work(new: np.ndarray, lengths: np.ndarray, heads: int, kv_heads: int, sms: int, head_dim: int = 64, form: int = -1) -> _Work:
    fn = _lib.rt_lib().apb_rt_kv8_plan
    c = ctypes
    fn.argtypes, fn.restype = [c.c_void_p, c.c_void_p, c.c_int32, c.c_int32, c.c_int32, c.c_int32, c.c_int32, c.c_int32, c.c_void_p, c.c_int64, c.c_void_p,
                               c.c_void_p, c.c_int64, c.c_void_p], c.c_int32
    new, lengths = np.ascontiguousarray(new, dtype=np.int32), np.ascontiguousarray(lengths, dtype=np.int32)
    counts, first = np.zeros(5, dtype=np.int64), np.zeros(sms + 1, dtype=np.int32)
    # the first call says how many there are
    items, joins = np.empty((0, 12), dtype=np.int32), np.empty((0, 8), dtype=np.int32)
    for _ in range(2):
        if fn(new.ctypes.data, lengths.ctypes.data, len(new), heads, kv_heads, head_dim, sms, form, items.ctypes.data, len(items), first.ctypes.data,
              joins.ctypes.data, len(joins), counts.ctypes.data) != 0:
            raise ValueError("chunk plan: sizes out of range")
        if len(items) >= counts[0] and len(joins) >= counts[1]:
            break
        items, joins = np.empty((int(counts[0]), 12), dtype=np.int32), np.empty((int(counts[1]), 8), dtype=np.int32)
    return _Work(items, first[:int(counts[3]) + 1], joins, int(counts[2]), int(counts[3]), int(counts[4]))


def _few(new: np.ndarray, lengths: np.ndarray, heads: int, kv_heads: int, sms: int, head_dim: int = 128) -> bool:
    """Whether the tokens are so few that they go the way of decode attention."""
    fn = _lib.rt_lib().apb_rt_kv8_few
    fn.argtypes, fn.restype = [ctypes.c_void_p] * 2 + [ctypes.c_int32] * 5, ctypes.c_int32
    new, lengths = np.ascontiguousarray(new, dtype=np.int32), np.ascontiguousarray(lengths, dtype=np.int32)
    return bool(fn(new.ctypes.data, lengths.ctypes.data, len(new), heads, kv_heads, head_dim, sms))


@dataclass
class ChunkPlan:
    """Tables of a step in which every sequence brings some tokens; made on the host once and used by all layers.  They go to the cache's
    device on the current stream.

    Sequence ``s`` has ``lengths[s]`` tokens in the cache, the last ``new[s]`` of which are its query rows (row ``i`` sees the tokens
    up to position ``lengths[s] - new[s] + i``; one below 0 sees nothing); the rows of the sequences follow one another."""
    rows: int
    new: np.ndarray
    lengths: np.ndarray
    pages: List[np.ndarray]
    heads: int
    kv_heads: int
    num_pages: int
    head_dim: int
    work: Optional[_Work] = None                     # None: few tokens of each sequence, the way of decode attention
    table: Optional[torch.Tensor] = None             # on the cache's device: pages, and the work's tables
    items: Optional[torch.Tensor] = None
    first: Optional[torch.Tensor] = None
    joins: Optional[torch.Tensor] = None
    # without work: the lengths [n], where the sequences' rows begin [n + 1], the most new tokens and pages of a sequence
    few: Optional[Tuple[torch.Tensor, torch.Tensor, int, int]] = None

    @staticmethod
    def build(new: Sequence[int], lengths: Sequence[int], pages, heads: int, cache: Fp8KVCache) -> "ChunkPlan":
        """``pages``: per sequence its page ids in order (a table's further entries are not looked at)."""
        new, lengths = np.asarray(new, dtype=np.int64).reshape(-1), np.asarray(lengths, dtype=np.int64).reshape(-1)
        n = len(new)
        if len(lengths) != n or len(pages) != n or (new < 0).any() or (lengths < 0).any():
            raise ValueError("new, lengths and pages describe the same sequences, with counts from 0 on")
        if heads < 1 or heads % cache.num_kv_heads:
            raise ValueError(f"{heads} query heads are not a multiple of {cache.num_kv_heads} key heads")
        if new.sum() >= 1 << 31 or (n and lengths.max() >= 1 << 31):
            raise ValueError("more rows or tokens than 2^31")
        need = (lengths + PAGE - 1) // PAGE
        used = []
        for s in range(n):
            p = np.asarray(pages[s]).reshape(-1)[:need[s]]
            if len(p) < need[s]:
                raise ValueError(f"sequence {s}: {len(p)} pages do not hold {lengths[s]} tokens")
            if len(p) and (p.min() < 0 or p.max() >= cache.num_pages):
                raise ValueError(f"sequence {s}: a page outside the cache's {cache.num_pages}")
            used.append(p.astype(np.int32))
        rows = int(new.sum())
        plan = ChunkPlan(rows, new, lengths, used, heads, cache.num_kv_heads, cache.num_pages, cache.head_dim)
        if cache.index >= 0 and rows:
            sms = torch.cuda.get_device_properties(cache.data.device).multi_processor_count
            sizes = (new, lengths, heads, cache.num_kv_heads, sms)
            if not _few(*sizes, cache.head_dim):
                plan.work = w = _work(*sizes, cache.head_dim)
            table = np.zeros((n, max(1, int(need.max()))), dtype=np.int32)
            for s in range(n):
                table[s, :need[s]] = used[s]
            if plan.work is None:
                parts = (table, lengths.astype(np.int32), np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
            else:
                parts = (w.items, w.joins, w.first, table)
            flat = torch.from_numpy(np.concatenate([a.reshape(-1) for a in parts])).pin_memory()
            dev = [t.view(a.shape) for t, a in zip(to_device(flat, cache.data.device).split([a.size for a in parts]), parts)]
            if plan.work is None:
                plan.table, plan.few = dev[0], (dev[1], dev[2], int(new.max()), int(need.max()))
            else:
                plan.items, plan.joins, plan.first, plan.table = dev
        return plan


def chunk_attention(q: torch.Tensor, cache: Fp8KVCache, plan: ChunkPlan, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``q [T, Hq, D]`` bf16, the new tokens of the plan's sequences one behind another -> ``[T, Hq, D]`` bf16.  Each row sees the
    tokens of its sequence up to itself (:class:`ChunkPlan`), rows that see nothing are zeros.  Rows of ``q`` behind the last
    sequence are padding: they are left as they were in ``out``, zeros without it.  The new tokens' own keys and values are read from the
    cache: :func:`write` comes first.  Rows of the cache whose exponents lie more than 100 below the largest of their sequence (values) or of
    their 128 tokens (keys) lose bits.
    A key that is no number reaches the rows that see it, such a value that column of its sequence's rows, those in front of it too.  A
    captured call reads the plan's tables when it is replayed: the plan has to live as long."""
    q, ldq = _check_queries(q, cache, out)
    data = cache.data
    T, Hq, D = q.shape
    if (Hq, cache.num_kv_heads, cache.num_pages, D) != (plan.heads, plan.kv_heads, plan.num_pages, plan.head_dim):
        raise ValueError("the plan was made for other heads or another cache")
    if T < plan.rows:
        raise ValueError(f"q has {T} rows, the plan's sequences bring {plan.rows}")
    scale = D ** -0.5 if scale is None else float(scale)
    if out is None:
        out = _rows(T, Hq, D, data, torch.bfloat16)
        if T > plan.rows:
            out[plan.rows:].zero_()
    if plan.rows == 0:
        return out
    if cache.index < 0:
        row = 0
        for m, n, p in zip(plan.new.tolist(), plan.lengths.tolist(), plan.pages):
            k, v = context_ref(cache, torch.from_numpy(p), n)
            out[row:row + m] = attention_ref(q[row:row + m].float(), k, v, torch.arange(n - m, n), scale).to(q.dtype)
            row += m
        return out
    if plan.table is None or plan.table.get_device() != cache.index:
        raise ValueError(f"the plan was not made for a cache on {data.device}")
    if out.stride(0) % 8 or out.data_ptr() % 16:             # rows off the 16-byte boundaries: by way of a copy
        out[:plan.rows].copy_(chunk_attention(q, cache, plan, scale)[:plan.rows])
        return out
    if _elsewhere(cache):
        with torch.cuda.device(cache.index):
            return chunk_attention(q, cache, plan, scale, out)
    w = plan.work
    if w is None:
        table, (lengths, starts, most, longest) = plan.table, plan.few
        _lib.check(_fn("few")(q.data_ptr(), ldq, data.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1], cache.num_pages,
                              lengths.data_ptr(), starts.data_ptr(), out.data_ptr(), out.stride(0), table.shape[0], most, longest, Hq,
                              cache.num_kv_heads, D, scale, _lib.stream_ptr()), "kv8_few")
        return out
    scratch = torch.empty(w.part_tiles * 128 * (D + 2), device=data.device, dtype=torch.float32) if w.part_tiles else None
    _lib.check(_fn("chunk")(q.data_ptr(), ldq, data.data_ptr(), plan.table.data_ptr(), plan.table.stride(0), plan.items.data_ptr(),
                            plan.first.data_ptr(), w.ctas, plan.joins.data_ptr(), len(w.joins), w.part_tiles, w.form, _lib.ptr(scratch),
                            out.data_ptr(), out.stride(0), T, Hq, cache.num_kv_heads, D, scale, _lib.stream_ptr()), "kv8_chunk")
    return out
