"""Tokens drawn from rows of logits with given random numbers.

``sample(logits, uniforms, temperature, top_k, top_p, min_p)`` draws one token per row.  Of a row of logits ``l`` at temperature ``T``

* the tokens stay whose logit is at least the ``top_k``-th largest, those with ``exp((l - max) / T) >= min_p``, and of what is left those of
  which the strictly larger ones hold less than ``top_p`` of its mass (equal logits stay or go together, the largest always stay);
* the token is the first one, in the order of the vocabulary, up to which, itself included, the mass of what stayed is above ``u``
  times all of it (a mass below e^-693 of the largest one's counts as none); at ``T <= 0`` the first of the largest logits, whatever the
  other settings are;
* its log-probability is that of ``softmax(l / T)`` without restrictions (of ``softmax(l)`` at ``T <= 0``), as a policy's gradient wants it.

The order of the restrictions is that of ``engine/reference_sampler.py``.  Masses are 64-bit numbers.  CUDA tensors run ``csrc/draw.cu``,
CPU tensors the expression below (the oracle of the GPU tests).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from . import _lib

MOST_VOCABULARY = 3 << 17
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_FN = None


def _fn():
    global _FN
    if _FN is None:
        c = ctypes
        vp, i, ll, f = c.c_void_p, c.c_int, c.c_longlong, c.c_float
        _FN = _lib.declare("apb_draw", [vp, i, ll, vp, f, vp, i, vp, f, vp, f, vp, i, c.c_uint, vp, vp, i, i, vp, vp, vp])
    return _FN


def draw_raw(logits: torch.Tensor, uniforms: Optional[torch.Tensor], temperature, top_k, top_p, min_p, tokens: torch.Tensor,
             logprobs: torch.Tensor, seed: Union[int, torch.Tensor] = 0, step: Optional[torch.Tensor] = None) -> None:
    """The launch behind :func:`sample` on checked arguments of the current device: each setting a number or a contiguous tensor ``[B]``
    (fp32, ``top_k`` int32).  Without ``uniforms`` the token is the largest of ``l / T`` and Gumbel noise by a hash of
    ``seed``, ``step``, the row and the token, the noise of the rollout engine's other draws; seed and step on the device (one int32 each)
    are read by the kernel, so that a captured graph sees new values."""
    both = lambda x, off: (None, x) if not torch.is_tensor(x) else (x.data_ptr(), off)          # noqa: E731
    _lib.check(_fn()(logits.data_ptr(), _TYPES[logits.dtype], logits.stride(0), *both(temperature, 1.0), *both(top_k, 0), *both(top_p, 1.0),
                     *both(min_p, 0.0), None if uniforms is None else uniforms.data_ptr(),
                     uniforms is not None and uniforms.dtype is torch.float64,
                     ctypes.c_uint(0 if torch.is_tensor(seed) else seed & 0xFFFFFFFF), seed.data_ptr() if torch.is_tensor(seed) else None,
                     None if step is None else step.data_ptr(), logits.shape[0], logits.shape[1], tokens.data_ptr(), logprobs.data_ptr(),
                     _lib.stream_ptr()), "apb_draw")


def sample_ref(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """:func:`sample` as an expression in 64 bits, on any device."""
    B, V = logits.shape
    if B == 0:
        return logits.new_zeros(0, dtype=torch.int32), logits.new_zeros(0, dtype=torch.float32)
    z = logits.double()
    z = torch.where(torch.isnan(z), float("-inf"), z)
    column = lambda x, dtype: torch.as_tensor(x, dtype=dtype, device=z.device).expand(B)[:, None]       # noqa: E731
    at = torch.arange(V, device=z.device)
    # settings are fp32 numbers in the kernel
    T, p, m = (column(x, torch.float32).double() for x in (temperature, top_p, min_p))
    k = column(top_k, torch.int64)
    greedy = ~(T > 0)
    T = torch.where(greedy, 1.0, T)
    most = z.amax(-1, keepdim=True)
    x = torch.where(z == most, 0.0, (z - torch.where(torch.isinf(most) & (most < 0), 0.0, most)) / T)
    full = torch.where(x < -693.0, 0.0, x.exp())
    order = torch.sort(z, dim=-1, descending=True).values
    kth = order.gather(1, torch.where((k > 0) & (k < V), k, V) - 1)
    keep = (z >= kth) & ((m <= 0) | torch.isnan(m) | (x >= torch.log(m.clamp_max(1.0))))
    mass = torch.where(keep, full, 0.0)
    value, rank = torch.sort(z, dim=-1, descending=True, stable=True)
    run = mass.gather(1, rank).cumsum(-1)
    value = -value.contiguous()
    first = torch.searchsorted(value, value)
    larger = torch.where(first > 0, run.gather(1, (first - 1).clamp_min(0)), 0.0)
    stays = (larger < p * run[:, -1:]) | ~(p < 1) | (value == -most)
    mass = torch.where(torch.zeros_like(keep).scatter(1, rank, stays), mass, 0.0)
    run = mass.cumsum(-1)
    u = torch.where(uniforms < 1, uniforms.double().clamp_min(0.0), 1 - 2.0 ** -52)[:, None]
    token = (run <= u * run[:, -1:]).sum(-1)
    token = torch.minimum(token, torch.where(mass > 0, at, 0).amax(-1))
    token = torch.where(greedy[:, 0], torch.where(z == most, at, V).amin(-1), token)
    logprob = x.gather(1, token[:, None])[:, 0] - full.sum(-1).log()
    nothing = torch.isinf(most[:, 0]) & (most[:, 0] < 0)
    return torch.where(nothing, 0, token).to(torch.int32), torch.where(nothing, float("-inf"), logprob).float()


Setting = Union[float, int, torch.Tensor]


def sample(logits: torch.Tensor, uniforms: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0,
           min_p: Setting = 0.0, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``logits [B, V]`` (fp32, bf16 or fp16; rows may be strided), ``uniforms [B]`` in [0, 1) (fp32 or fp64) -> ``(tokens [B] int32,
    logprobs [B] fp32)``.  Each setting is a number or a tensor ``[B]`` (``top_k`` of integers): ``temperature`` <= 0 takes the largest
    logit, ``top_k`` <= 0 or of V and more, ``top_p`` >= 1 and ``min_p`` <= 0 are off.  ``out``: contiguous int32 and fp32 tensors
    ``[B]`` that take the result.

    Logits that are not numbers are never drawn; in a row without any above ``-inf`` token 0 comes out, with log-probability ``-inf``.
    A uniform below 0 counts as 0, one of 1 or more, or that is not a number, as the largest number below 1."""
    if logits.dim() != 2 or logits.dtype not in _TYPES or logits.shape[1] < 1:
        raise ValueError(f"logits must be fp32, bf16 or fp16 [B, V], got {logits.dtype} {list(logits.shape)}")
    B, V = logits.shape
    if uniforms.dtype not in (torch.float32, torch.float64) or uniforms.shape != (B,):
        raise ValueError(f"uniforms must be fp32 or fp64 [{B}], got {uniforms.dtype} {list(uniforms.shape)}")
    on = logits.device
    for name, x in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        if torch.is_tensor(x):
            if x.shape != (B,) or x.device != on:
                raise ValueError(f"{name} must be a number or [{B}] on {on}, got {list(x.shape)} on {x.device}")
            if x.is_floating_point() == (name == "top_k") or x.dtype is torch.bool or x.is_complex():
                raise ValueError(f"{name} cannot be {x.dtype}")
    if uniforms.device != on:
        raise ValueError(f"uniforms live on {uniforms.device}, logits on {logits.device}")
    if out is not None:
        for name, t, dtype in (("out[0]", out[0], torch.int32), ("out[1]", out[1], torch.float32)):
            if t.shape != (B,) or t.dtype != dtype or not t.is_contiguous() or t.device != on:
                raise ValueError(f"{name} must be contiguous {dtype} [{B}] on {on}, got {t.dtype} {list(t.shape)} on {t.device}")
    if not logits.is_cuda:
        tokens, logprobs = sample_ref(logits, uniforms, temperature, top_k, top_p, min_p)
        if out is None:
            return tokens, logprobs
        out[0].copy_(tokens)
        out[1].copy_(logprobs)
        return out[0], out[1]
    if V > MOST_VOCABULARY:
        raise ValueError(f"rows of {V} logits: at most {MOST_VOCABULARY} are drawn from on a GPU")
    if logits.get_device() != torch._C._cuda_getDevice():
        with torch.cuda.device(logits.device):
            return sample(logits, uniforms, temperature, top_k, top_p, min_p, out)
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    # the usual types pass as they are: a conversion that converts nothing still costs the host a microsecond
    whole = lambda x, dtype: x if x.dtype is dtype and x.is_contiguous() else x.to(dtype).contiguous()      # noqa: E731
    number = lambda x: whole(x, torch.float32) if torch.is_tensor(x) else float(x)                            # noqa: E731
    if torch.is_tensor(top_k):
        top_k = whole(top_k.clamp(0, V) if top_k.dtype is torch.int64 else top_k, torch.int32)
    else:
        top_k = max(0, min(int(top_k), V))
    tokens, logprobs = out if out is not None else (torch.empty(B, device=on, dtype=torch.int32), torch.empty(B, device=on, dtype=torch.float32))
    draw_raw(logits, uniforms if uniforms.is_contiguous() else uniforms.contiguous(), number(temperature), top_k, number(top_p), number(min_p), tokens, logprobs)
    return tokens, logprobs
