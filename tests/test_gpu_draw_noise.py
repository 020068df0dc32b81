"""The noise of draws without given numbers: -log(-log(x)) of a uniform x that a hash of seed, step, row and token gives.

x lies in the middle of one of 2^24 steps, so that the largest noise is -log(-log(1 - 2^-25)) = 17.4 and a token 40 below the largest
logit cannot win: the largest one's own noise is at least -log(-log(2^-25)) = -2.9, which leaves 37 between them."""
import ctypes

import pytest
import torch

from arctic_platform_b200.engine.sampler import _fn
from arctic_platform_b200.ops import _lib, sampling

# (seed, step, row, token) whose hash begins with 24 ones
LARGEST = [(99, 0, 95, 120745), (1, 1, 2, 131890), (7, 8, 7, 17072)]
MASK = (1 << 32) - 1


def _hash(x):
    x = x ^ (x >> 16)
    x = x * 0x7FEB352D & MASK
    x = x ^ (x >> 15)
    x = x * 0x846CA68B & MASK
    return x ^ (x >> 16)


def leading(seed, step, row, tokens):
    """The 24 leading bits of the hash of ``tokens`` (an int, or an int64 tensor)."""
    base = _hash(seed ^ (step * 0x9E3779B9 & MASK)) ^ _hash((row * 0x85EBCA6B & MASK) + 1 & MASK)
    return _hash(base + tokens * 0x9E3779B9 & MASK) >> 8


def test_the_named_tokens_have_the_largest_uniform():
    for seed, step, row, token in LARGEST:
        assert leading(seed, step, row, token) == (1 << 24) - 1


def draw(how, z, seed, step):
    B, V = z.shape
    out = torch.empty(B, device="cuda", dtype=torch.int32), torch.empty(B, device="cuda")
    one = torch.ones(B, device="cuda")
    at = torch.full((1,), step, device="cuda", dtype=torch.int32)
    if how == "engine":
        _lib.check(_fn("sample")(_lib.ptr(z), z.stride(0), _lib.ptr(one), B, V, ctypes.c_uint(seed), _lib.ptr(at), _lib.ptr(out[0]),
                                 _lib.ptr(out[1]), _lib.stream_ptr()), "sample")
    elif how == "engine, top-k":
        topk, topp, thr = torch.full((B,), V - 1, device="cuda", dtype=torch.int32), one, torch.empty(B, device="cuda")
        _lib.check(_fn("sample_f")(_lib.ptr(z), z.stride(0), _lib.ptr(one), B, V, ctypes.c_uint(seed), _lib.ptr(at), _lib.ptr(topk),
                                   _lib.ptr(topp), _lib.ptr(thr), _lib.ptr(out[0]), _lib.ptr(out[1]), _lib.stream_ptr()), "sample_f")
    else:
        sampling.draw_raw(z, None, 1.0, 0, 1.0, 1e-30 if how == "min-p" else 0.0, *out, seed=seed, step=at)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["engine", "engine, top-k", "raw", "min-p"])
@pytest.mark.parametrize("where", LARGEST)
def test_an_unlikely_token_is_not_drawn_for_its_noise(how, where):
    seed, step, row, token = where
    V = token + 1001
    z = torch.zeros((row + 1, V), device="cuda")
    z[:, token] = -40.0
    z[:, 0] = -60.0                            # the one that top-k leaves out
    tokens, _ = draw(how, z, seed, step)
    assert int(tokens[row]) != token


@pytest.mark.gpu
def test_the_largest_uniform_has_a_finite_noise():
    """At equal logits the token with the largest uniform still is the one that is drawn."""
    for seed, step, row, token in LARGEST:
        z = torch.zeros((row + 1, token + 1001), device="cuda")
        for how in ("engine", "raw"):
            assert int(draw(how, z, seed, step)[0][row]) == token
