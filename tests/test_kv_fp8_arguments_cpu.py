"""Arguments of the 8-bit cache's operators that a kernel would take on trust: what is refused on the host, without a GPU."""
import threading

import pytest
import torch

from arctic_platform_b200.ops import kv_fp8

H, D, B, HEADS = 2, 64, 3, 4


def _step(**other):
    cache = kv_fp8.Fp8KVCache.zeros(4, H, D, device="cpu")
    a = dict(acc=torch.zeros(B, (HEADS + 2 * H) * D), q_norm=torch.ones(D).bfloat16(), k_norm=torch.ones(D).bfloat16(),
             rope=(torch.ones(9, D // 2), torch.zeros(9, D // 2)), positions=torch.zeros(B, dtype=torch.int32),
             slots=torch.arange(B, dtype=torch.int32), cache=cache, heads=HEADS, eps=1e-6)
    return {**a, **other}


@pytest.mark.parametrize("what,other,message", [
    ("fewer sines than cosines", dict(rope=(torch.ones(9, D // 2), torch.zeros(8, D // 2))), "sin"),
    ("angles in three dimensions", dict(rope=(torch.ones(1, 9, D // 2), torch.zeros(1, 9, D // 2))), "cos"),
    ("a weight per head", dict(q_norm=torch.ones(HEADS, D).bfloat16()), "q_norm"),
    ("a weight of another size", dict(k_norm=torch.ones(2 * D).bfloat16()), "k_norm"),
    ("a weight in fp32", dict(k_norm=torch.ones(D)), "k_norm"),
    ("no query heads", dict(acc=torch.zeros(B, 2 * H * D), heads=0), "acc"),
    ("rows of sums over one another", dict(acc=torch.zeros(1, (HEADS + 2 * H) * D).expand(B, -1)), "acc"),
])
def test_a_steps_arguments_are_refused(what, other, message):
    with pytest.raises(ValueError, match=message):
        kv_fp8.norm_rope_write(**_step(**other))


def test_a_step_asks_where_each_of_its_tensors_lives(monkeypatch):
    """Their addresses go to the kernel: one in host memory would be an illegal access."""
    seen = set()
    monkeypatch.setattr(kv_fp8, "_refuse", lambda cache, **t: seen.update(t))
    with pytest.raises(ValueError, match="runs on a GPU"):
        kv_fp8.norm_rope_write(**_step())
    assert seen >= {"acc", "positions", "cos", "sin", "q_norm", "k_norm"}


def test_queries_that_share_their_memory_get_rows_of_their_own():
    cache = kv_fp8.Fp8KVCache.zeros(4, H, D, device="cpu")
    one = torch.randn(1, HEADS, D).bfloat16()
    q, distance = kv_fp8._check_queries(one.expand(5, -1, -1), cache, None)
    assert distance == q.stride(0) == HEADS * D and torch.equal(q, one.expand(5, -1, -1))
    over = torch.zeros(5 * 8 + HEADS * D).bfloat16().as_strided((5, HEADS, D), (8, D, 1))
    assert kv_fp8._check_queries(over, cache, None)[1] == HEADS * D
    wide = torch.zeros(5, 3 * HEADS, D).bfloat16()[:, HEADS:2 * HEADS]
    assert kv_fp8._check_queries(wide, cache, None)[0] is wide                # rows of their own stay where they are


@pytest.mark.parametrize("what", ["decode", "chunk"])
def test_outputs_over_one_another_are_refused(what):
    cache = kv_fp8.Fp8KVCache.zeros(4, H, D, device="cpu")
    q, table, n = torch.zeros(B, HEADS, D).bfloat16(), torch.zeros(B, 1, dtype=torch.int32), torch.ones(B, dtype=torch.int32)
    plan = kv_fp8.ChunkPlan.build([1] * B, [1] * B, table.numpy(), HEADS, cache)
    for out in (q[:1].clone().expand(B, -1, -1), torch.zeros(2 * 64 + HEADS * D).bfloat16().as_strided((B, HEADS, D), (64, D, 1))):
        with pytest.raises(ValueError, match="out must"):
            kv_fp8.decode_attention(q, cache, table, n, out=out) if what == "decode" else kv_fp8.chunk_attention(q, cache, plan, out=out)
    one = q[:1].clone().expand(B, -1, -1)[:1]                                    # a single row has no neighbour
    kv_fp8.decode_attention(q[:1], cache, table[:1], n[:1], out=one)


def test_two_threads_may_make_the_first_call(monkeypatch):
    """The table of the kernels' entry points is there as a whole or not at all."""
    monkeypatch.setattr(kv_fp8, "_FN", {})
    half_way, go_on = threading.Event(), threading.Event()

    def declare(name, *types):
        if threading.current_thread() is first and name == "apb_kv8_read":
            half_way.set()
            go_on.wait(10)
        return name

    monkeypatch.setattr(kv_fp8._lib, "declare", declare)
    first = threading.Thread(target=lambda: kv_fp8._fn("write"))
    first.start()
    try:
        assert half_way.wait(10)
        assert kv_fp8._fn("chunk") == "apb_kv8_chunk"
    finally:
        go_on.set()
        first.join()
    assert kv_fp8._fn("write") == "apb_kv8_write"


def test_sequences_that_are_not_active_are_empty():
    cache = kv_fp8.Fp8KVCache.zeros(4, H, D, device="cpu")
    g = torch.Generator().manual_seed(0)
    kv_fp8.write(*(torch.randn(40, H, D, generator=g) for _ in range(2)), torch.arange(40, dtype=torch.int32), cache)
    q = torch.randn(B, HEADS, D, generator=g).bfloat16()
    table, n = torch.arange(3, dtype=torch.int32).expand(B, 3), torch.tensor([40, 33, 7], dtype=torch.int32)
    active = torch.tensor([1, 0, 2], dtype=torch.int32)
    want = kv_fp8.decode_attention(q, cache, table, n * (active > 0))
    assert torch.equal(kv_fp8.decode_attention(q, cache, table, n, active=active), want) and not want[1].any() and want[0].any()
    for bad in (active.long(), active[:2], active.expand(B, B), torch.zeros(2 * B, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="active must"):
            kv_fp8.decode_attention(q, cache, table, n, active=bad)


@pytest.mark.parametrize("asked,head_dim,served,reported", [
    ("fp8", 128, "fp8", False), ("fp8_e4m3", 64, "fp8_e4m3", False), ("auto", 256, None, False), (None, 256, None, False), ("bfloat16", 128, None, False),
    ("fp8_e5m2", 128, None, True), ("int8", 64, None, True), ("fp8", 256, None, True), ("fp8", 96, None, True), ("fp8", None, None, False)])
def test_cache_types_that_are_not_served_are_reported(caplog, asked, head_dim, served, reported):
    from arctic_platform_b200.engine.hybrid_sampler import HybridSampler
    from arctic_platform_b200.engine.sampler import SamplerEngine
    from arctic_platform_b200.engine.worker import EngineWorker
    assert EngineWorker._kv_cache_dtype(SamplerEngine, {"kv_cache_dtype": asked}, head_dim) == {"kv_cache_dtype": served}
    assert bool(caplog.records) == reported and all(repr(asked) in r.getMessage() for r in caplog.records)
    caplog.clear()
    assert EngineWorker._kv_cache_dtype(HybridSampler, {"kv_cache_dtype": asked}, head_dim) == {}
    assert bool(caplog.records) == (reported or served is not None)


@pytest.mark.parametrize("asked", ["fp8", "fp8_e5m2", "nonsense"])
def test_a_job_whose_cache_type_is_not_served_runs(asked, caplog):
    from arctic_platform_b200.rl import ArcticRLClientConfig, create_arctic_rl_client
    client = create_arctic_rl_client(ArcticRLClientConfig(
        comm_protocol="local", model_name="qwen3-tiny", training_gpus=1, sampling_gpus=1, colocate=True,
        ds_config={"optimizer": {"params": {"lr": 1e-4}}}, vllm_config={"max_num_seqs": 4, "max_model_len": 64, "kv_cache_dtype": asked}))
    client.call("sync_weights")
    out = client.call("generate", [[1, 2, 3]], {"n": 1, "temperature": 0.0, "max_tokens": 2, "ignore_eos": True})
    assert len(out[0]["token_ids"]) == 2 and repr(asked) in caplog.text


def test_a_draft_models_engine_says_that_it_has_no_8_bit_cache(caplog):
    from arctic_platform_b200.rl import ArcticRLClientConfig, create_arctic_rl_client
    client = create_arctic_rl_client(ArcticRLClientConfig(
        comm_protocol="local", model_name="qwen3-tiny", training_gpus=1, sampling_gpus=1, colocate=True,
        ds_config={"optimizer": {"params": {"lr": 1e-4}}}, vllm_config={"max_num_seqs": 4, "max_model_len": 64, "kv_cache_dtype": "fp8"},
        arctic_inference_config={"speculative_decoding": {"model": "qwen3-tiny", "num_speculative_tokens": 2}}))
    assert len(client.call("generate", [[1, 2, 3]], {"n": 1, "temperature": 0.0, "max_tokens": 2, "ignore_eos": True})[0]["token_ids"]) == 2
    assert "SpeculativeSampler" in caplog.text and "'fp8'" in caplog.text
