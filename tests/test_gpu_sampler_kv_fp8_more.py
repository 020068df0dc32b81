"""The rollout engine on the 8-bit cache: sequences that have ended, every step of a rollout, experts, 8-bit weights, scoring."""
import numpy as np
import pytest
import torch

from tests.test_gpu_sampler_kv_fp8 import _engine

pytestmark = pytest.mark.gpu


def test_sequences_that_have_ended_are_not_read(monkeypatch):
    """Between two harvests their lengths are still there; the steps pass on which slots are active."""
    from arctic_platform_b200.ops import kv_fp8
    model, eng = _engine(kv_cache_dtype="fp8", use_cuda_graph=False, sync_interval=16)
    plain, ended = kv_fp8.decode_attention, []

    def spy(q, cache, table, lengths, *a, active=None, **kw):
        out = plain(q, cache, table, lengths, *a, active=active, **kw)
        over = (lengths > 0) & (active <= 0)
        ended.append((int(over.sum()), bool(out[over].any())))
        return out

    monkeypatch.setattr(kv_fp8, "decode_attention", spy)
    prompts = [list(range(5, 45)), list(range(7, 30)), list(range(90, 200))]
    free = [o["token_ids"] for o in eng.generate(prompts, {"temperature": 0.0, "max_tokens": 40})]
    # a token that ends one sequence within a few steps and another one late or never
    first = {t: [next((i for i, x in enumerate(o) if x == t), 99) for o in free] for o in free for t in o[1:12]}
    stop = max(first, key=lambda t: max(first[t]) - min(first[t]))
    assert max(first[stop]) - min(first[stop]) > 2
    ended.clear()
    out = eng.generate(prompts, {"temperature": 0.0, "max_tokens": 40, "stop_token_ids": [stop]})
    assert [len(o["token_ids"]) < 40 for o in out] == [f < 39 for f in first[stop]]
    assert any(n for n, _ in ended) and not any(some for _, some in ended)
