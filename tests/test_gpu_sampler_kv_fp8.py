"""The rollout engine on the 8-bit cache: what a step writes, what it attends to, whole rollouts against an engine on bf16 keys and values
that hold the same numbers."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _engine(preset="qwen3-tiny-d128", model=None, **kw):
    from arctic_platform_b200.engine.sampler import SamplerEngine
    from arctic_platform_b200.models.config import PRESETS
    from arctic_platform_b200.models.decoder import DecoderLM
    cfg = PRESETS[preset]
    model = model or DecoderLM(cfg, "cuda", torch.bfloat16).init_weights(seed=5, std=0.05)
    kw = {"kv_cache_tokens": 1 << 14, "max_batch": 16, "max_seq_len": 512, "sync_interval": 4, **kw}
    return model, SamplerEngine(cfg, "cuda", model=model, **kw)


@pytest.mark.parametrize("Hq,H,D,B,norm", [(32, 8, 128, 7, True), (4, 2, 64, 3, True), (5, 1, 128, 1, False), (16, 8, 64, 130, False)])
def test_a_steps_projection_is_normed_rotated_and_written(Hq, H, D, B, norm):
    """Codes, exponents and q are those of the bf16 epilogue followed by a write of its rows."""
    from arctic_platform_b200.engine.sampler import _fn
    from arctic_platform_b200.ops import _lib, kv_fp8
    g = torch.Generator(device="cuda").manual_seed(B)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    acc = r(B, (Hq + 2 * H) * D + 32)[:, :(Hq + 2 * H) * D]
    wq, wk = (r(D).bfloat16(), r(D).bfloat16()) if norm else (None, None)
    angle = r(50, D // 2)
    rope = angle.cos().contiguous(), angle.sin().contiguous()
    pos = torch.randint(0, 50, (B,), device="cuda", generator=g, dtype=torch.int32)
    pages = B // 16 + 2
    slots = torch.randperm(pages * 16, device="cuda", generator=g)[:B].to(torch.int32)
    slots[B // 2] = -1
    sums = acc.clone()
    q = torch.empty((B, Hq, D), device="cuda", dtype=torch.bfloat16)
    kc, vc = (torch.zeros((pages, H, 16, D), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    _lib.check(_fn("qkv_post")(_lib.ptr(sums), sums.stride(0), _lib.ptr(wq), _lib.ptr(wk), _lib.ptr(rope[0]), _lib.ptr(rope[1]), _lib.ptr(pos),
                               _lib.ptr(slots), _lib.ptr(q), _lib.ptr(kc), _lib.ptr(vc), B, Hq, H, D, 1e-6, _lib.stream_ptr()), "qkv_post")
    page, t = slots.long().clamp_min(0) // 16, slots.long().clamp_min(0) % 16
    want = kv_fp8.Fp8KVCache.zeros(pages, H, D)
    kv_fp8.write(kc[page, :, t], vc[page, :, t], slots, want)
    got = kv_fp8.Fp8KVCache.zeros(pages, H, D)
    again = kv_fp8.norm_rope_write(acc, wq, wk, rope, pos, slots, got, Hq, 1e-6)
    assert torch.equal(again, q) and torch.equal(got.data, want.data) and not acc.any()
    with pytest.raises(ValueError):
        kv_fp8.norm_rope_write(acc[:, 1:], wq, wk, rope, pos, slots, got, Hq, 1e-6)
    with pytest.raises(ValueError):
        kv_fp8.norm_rope_write(acc, wq, wk, rope, pos.long(), slots, got, Hq, 1e-6)


def _same_numbers_in_bf16(eng):
    """Lets a bf16 engine hold what the 8-bit cache would."""
    from arctic_platform_b200.ops import kv_fp8
    plain = eng._write_kv

    def write(li, k, v, slots):
        c = kv_fp8.Fp8KVCache.zeros(k.shape[0] // 16 + 1, k.shape[1], k.shape[2])
        at = torch.arange(k.shape[0], device="cuda", dtype=torch.int32)
        kv_fp8.write(k, v, at, c)
        plain(li, *kv_fp8.read(c, at), slots)
    eng._write_kv = write


@pytest.mark.parametrize("graph", [False, True])
def test_rollouts_are_those_of_the_same_numbers_in_bf16(graph):
    """Greedy rollouts of several samples, more than there are slots.  Both engines attend to the same numbers; their attention rounds
    weights differently (fp16, bf16), so log-probabilities agree as those of two bf16 paths do, until a token differs."""
    from arctic_platform_b200.ops import _lib
    model, eng = _engine(kv_cache_dtype="fp8", use_cuda_graph=graph, split_k=False)
    _, other = _engine(model=model, use_cuda_graph=False, split_k=False, cascade=False)
    _same_numbers_in_bf16(other)
    rng = np.random.default_rng(0)
    prompts = [rng.integers(1, eng.cfg.vocab_size, size=n).tolist() for n in (37, 64, 5, 130, 16, 1)]
    sp = {"n": 3, "temperature": 0.0, "max_tokens": 21}
    a, b = eng.generate(prompts, sp), other.generate(prompts, sp)
    _lib.check_status("generate")
    assert eng.pages.free_count() == eng.num_pages
    compared = 0
    for x, y in zip(a, b):
        # up to the first token that differs, and that one: where all log-probabilities are within d of one another, so are the largest
        # ones, whichever token has them
        n = 1 + next((i for i, (s, t) in enumerate(zip(x["token_ids"], y["token_ids"])) if s != t), 20)
        assert n > 1                     # the first token comes from the prompt, which both attend to in bf16
        compared += n
        d = np.abs(np.array(x["logprobs"][:n]) - np.array(y["logprobs"][:n]))
        assert (d < 0.08).all() and d.mean() < 0.02
    assert compared >= 2 * len(a)
    assert len(a) == 18 and all(len(o["token_ids"]) == 21 for o in a)
    again = eng.generate(prompts, sp)
    assert [o["token_ids"] for o in again] == [o["token_ids"] for o in a]


def test_split_projection_and_small_heads():
    """The fused epilogue of the split-K projection in whole rollouts; a model of 64-wide heads; sleep and wake."""
    from arctic_platform_b200.ops import _lib
    for preset in ("qwen3-tiny-d128", "qwen3-tiny"):
        model, eng = _engine(preset, kv_cache_dtype="fp8_e4m3")
        _, plain = _engine(preset, model=model, kv_cache_dtype="fp8", split_k=False, use_cuda_graph=False)
        rng = np.random.default_rng(1)
        prompts = [rng.integers(1, eng.cfg.vocab_size, size=n).tolist() for n in (40, 9)]
        sp = {"n": 4, "temperature": 0.0, "max_tokens": 17}
        a, b = eng.generate(prompts, sp), plain.generate(prompts, sp)
        for x, y in zip(a, b):           # the first token comes from the prompt, the second from the first step
            assert x["token_ids"][0] == y["token_ids"][0] and abs(x["logprobs"][0] - y["logprobs"][0]) < 1e-3
            if x["token_ids"][1] == y["token_ids"][1]:
                assert abs(x["logprobs"][1] - y["logprobs"][1]) < 0.08
        eng.sleep()
        eng.wake()
        assert [o["token_ids"] for o in eng.generate(prompts, sp)] == [o["token_ids"] for o in a]
        _lib.check_status("generate")


def test_half_the_memory():
    model, eng = _engine(kv_cache_dtype="fp8")
    _, plain = _engine(model=model, kv_cache_dtype="auto")
    assert eng.num_pages == plain.num_pages and 0.5 < eng.kv_bytes() / plain.kv_bytes() < 0.51
    assert eng.kcache.numel() * eng.kcache.element_size() == eng.kv_bytes()


def test_refusals():
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        _engine(kv_cache_dtype="fp8_e5m2")
    with pytest.raises(NotImplementedError):
        _engine(kv_cache_dtype="fp8", tp_group=object())


def test_client_option_reaches_the_engine():
    from arctic_platform_b200.rl import ArcticRLClientConfig, create_arctic_rl_client
    client = create_arctic_rl_client(ArcticRLClientConfig(
        comm_protocol="local", model_name="qwen3-tiny-d128", training_gpus=1, sampling_gpus=1, colocate=True,
        ds_config={"optimizer": {"params": {"lr": 1e-4}}},
        vllm_config={"kv_cache_tokens": 1 << 13, "max_num_seqs": 8, "max_model_len": 256, "kv_cache_dtype": "fp8"}))
    client.call("sync_weights")
    out = client.call("generate", [list(range(5, 40))], {"n": 2, "temperature": 1.0, "max_tokens": 6, "ignore_eos": True})
    assert len(out) == 2 and all(len(o["token_ids"]) == 6 for o in out)
