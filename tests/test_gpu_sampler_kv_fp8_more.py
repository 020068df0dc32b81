"""The rollout engine on the 8-bit cache: sequences that have ended, every step of a rollout, experts, 8-bit weights, scoring."""
import numpy as np
import pytest
import torch

from tests.test_gpu_sampler_kv_fp8 import _engine, _same_numbers_in_bf16

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


def _force(eng, tokens):
    """Every slot is fed ``tokens [slots, steps]`` whatever it would choose; returns the logits that it chose from, by step."""
    plain, seen = eng._decode_logits, []

    def logits(B):
        out = plain(B)
        seen.append(out.clone())
        out.zero_().scatter_(1, tokens[:B, min(len(seen), tokens.shape[1]) - 1, None], 60.0)
        return out

    eng._decode_logits = logits
    return seen


@pytest.mark.parametrize("preset,quantization", [("qwen3-tiny-d128", None), ("qwen3-moe-tiny", None), ("tiny-fp8", "fp8")])
def test_every_step_of_rollouts_that_are_fed_the_same_tokens(monkeypatch, preset, quantization):
    """An engine on the 8-bit cache beside one that holds the same numbers in bf16, past several borders of pages.

    The first layer's keys and values depend on the fed tokens alone: what the cache holds of them is equal to the last bit, for every slot of
    every page.  Logits of the dense models differ by roundings: of the weights (2^-8) and of the output (2^-8 in either engine) of attention,
    and in each engine of about six tensors of a layer behind it whose roundings no longer agree, 15 * 2^-8 of the norm for each of two layers
    at most.  (Experts and 8-bit activations are chosen by such roundings: there no bound follows, and none is asked for.)"""
    import dataclasses

    from arctic_platform_b200.models import config
    from arctic_platform_b200.ops import _lib, kv_fp8
    if preset == "tiny-fp8":
        monkeypatch.setitem(config.PRESETS, preset, dataclasses.replace(config.PRESETS["qwen3-tiny-d128"], intermediate_size=768, name=preset))
    kw = {"use_cuda_graph": False, "split_k": False, "quantization": quantization}
    model, eng = _engine(preset, kv_cache_dtype="fp8", **kw)
    _, other = _engine(preset, model=model, cascade=False, **kw)
    _same_numbers_in_bf16(other)
    steps, rng = 36, np.random.default_rng(0)
    tokens = torch.from_numpy(rng.integers(1, eng.cfg.vocab_size, size=(16, steps))).cuda()
    prompts = [rng.integers(1, eng.cfg.vocab_size, size=n).tolist() for n in (37, 64, 5, 130, 16)]
    sp = {"n": 3, "temperature": 0.0, "max_tokens": steps, "ignore_eos": True}
    logits = [_force(e, tokens) for e in (eng, other)]
    a, b = eng.generate(prompts, sp), other.generate(prompts, sp)
    _lib.check_status("generate")
    assert [o["token_ids"] for o in a] == [o["token_ids"] for o in b] and all(len(o["token_ids"]) == steps for o in a)
    at = torch.arange(eng.num_pages * 16, device="cuda", dtype=torch.int32)
    page, t = at.long() // 16, at.long() % 16
    k, v = kv_fp8.read(eng._kv8[0], at)
    assert k.any() and torch.equal(k, other.kcache[0][page, :, t]) and torch.equal(v, other.vcache[0][page, :, t])
    assert all(torch.isfinite(x).all() for x in logits[0])
    if eng.cfg.is_moe or quantization:
        return
    for x, y in zip(*(seen[:steps - 1] for seen in logits)):
        x, y = x[:15].double(), y[:15].double()
        assert ((x - y).norm(dim=1) <= eng.cfg.num_layers * 15 * 2.0 ** -8 * y.norm(dim=1)).all()


def test_a_job_that_scores_takes_no_notice_of_the_cache_type():
    from arctic_platform_b200.engine.worker import EngineWorker
    prompts, completions = [[5, 6, 7, 8], [9, 10, 11]], [[12, 13, 14], [15, 16]]
    rows = []
    for vc in ({}, {"kv_cache_dtype": "fp8"}, {"kv_cache_dtype": "fp8_e5m2"}):
        w = EngineWorker()
        assert w.initialize({"job_type": "log_prob", "log_prob_engine": "vllm", "model_name": "qwen3-tiny-d128", "seed": 3, "vllm_config": vc})
        assert not w.sampler.kv_fp8
        rows.append(w.score_completions(prompts, completions))
    assert rows[0] == rows[1] == rows[2]
