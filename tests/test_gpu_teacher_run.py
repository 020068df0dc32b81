"""The operators around the output distribution as they are used together on a GPU: rollouts drawn with min_p, a teacher that answers its most likely
tokens, a student that learns from them; and the engines' part of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def engine(graph=True, **kw):
    from arctic_platform_b200.engine.sampler import SamplerEngine
    from arctic_platform_b200.models.config import PRESETS
    from arctic_platform_b200.models.decoder import DecoderLM
    cfg = PRESETS["qwen3-tiny-d128"]
    model = DecoderLM(cfg, "cuda", torch.bfloat16).init_weights(seed=5, std=0.05)
    return cfg, model, SamplerEngine(cfg, "cuda", model=model, kv_cache_tokens=1 << 14, max_batch=16, max_seq_len=512, sync_interval=4,
                                     use_cuda_graph=graph, **kw)


@pytest.mark.parametrize("graph", [False, True])
def test_min_p_in_the_paged_engine(graph):
    cfg, model, eng = engine(graph)
    prompts = [list(range(10, 40)), list(range(100, 117))]
    ask = {"n": 4, "temperature": 1.0, "max_tokens": 13, "seed": 3}
    greedy = eng.generate(prompts, {"n": 4, "temperature": 0.0, "max_tokens": 13})
    sure = eng.generate(prompts, {**ask, "min_p": 1.0})                  # only the most likely token is left
    assert [o["token_ids"] for o in sure] == [o["token_ids"] for o in greedy]
    a, b = eng.generate(prompts, {**ask, "min_p": 0.02}), eng.generate(prompts, {**ask, "min_p": 0.02})
    assert [o["token_ids"] for o in a] == [o["token_ids"] for o in b]    # a seed repeats
    c = eng.generate(prompts, {**ask, "min_p": 0.02, "seed": 4})         # another one does not, captured or not
    assert [o["token_ids"] for o in a] != [o["token_ids"] for o in c]
    assert len({tuple(o["token_ids"]) for o in a}) > 4
    # every drawn token has at least 0.02 of the most likely one's probability, and the log-prob of the unrestricted distribution
    from arctic_platform_b200.models.decoder import top_token_logprobs
    from arctic_platform_b200.ops.attention import AttnLayout
    import numpy as np
    for o in a[:5]:
        seq = prompts[o["prompt_index"]] + o["token_ids"]
        ids = torch.tensor(seq, device="cuda")
        with torch.no_grad():
            h = model.forward_hidden(ids, torch.arange(len(seq), device="cuda"), AttnLayout.from_cu_seqlens(np.array([0, len(seq)])))
        rows = h[o["prompt_len"] - 1:-1]
        best, _, _ = top_token_logprobs(model, rows, 1)
        lp = torch.tensor(o["logprobs"], device="cuda")
        assert bool((lp >= best[:, 0] + torch.log(torch.tensor(0.02)) - 0.1).all())      # the step's bf16 hidden states against the pass's
    plain = eng.generate(prompts, ask)
    again = eng.generate(prompts, {**ask, "min_p": 0.0})
    assert [o["token_ids"] for o in plain] == [o["token_ids"] for o in again]
    both = eng.generate(prompts, {**ask, "min_p": 0.01, "top_k": 3, "top_p": 0.9})
    assert len(both) == 8


def test_scores_with_their_most_likely_tokens():
    from arctic_platform_b200.engine.worker import EngineWorker
    w = EngineWorker("cuda:0")
    w.initialize({"model_name": "qwen3-tiny-d128", "job_type": "log_prob", "seed": 2})
    prompts, completions = [[5, 6, 7], [8, 9]], [[10, 11, 12], [13]]
    out = w.score_completions(prompts, completions, top_k=5)
    model = w._target_model()
    from arctic_platform_b200.ops.attention import AttnLayout
    import numpy as np
    for p, c, top in zip(prompts, completions, out["top_log_probs"]):
        ids = torch.tensor(p + c, device="cuda")
        with torch.no_grad():
            h = model.forward_hidden(ids, torch.arange(len(ids), device="cuda"), AttnLayout.from_cu_seqlens(np.array([0, len(ids)])))
        z = torch.log_softmax(h.float() @ model.output_weight.float().t(), -1)[len(p) - 1:-1]
        assert len(top) == len(c)
        for row, d in zip(z, top):
            v, i = row.topk(5)
            assert list(d) == i.tolist() and torch.allclose(torch.tensor(list(d.values())), v.cpu(), atol=3e-2)


def test_on_policy_distillation_from_rollout_to_step():
    from arctic_platform_b200.ops import _lib
    from arctic_platform_b200.rl import ArcticRLClientConfig, create_arctic_rl_client
    P, R, n_prompts, n = 24, 16, 3, 4
    client = create_arctic_rl_client(ArcticRLClientConfig(
        comm_protocol="local", model_name="qwen3-tiny-d128", training_gpus=1, sampling_gpus=1, log_prob_gpus=1, colocate=True, seed=3,
        ds_config={"zero_optimization": {"stage": 2}, "gradient_clipping": 1.0, "optimizer": {"type": "AdamW", "params": {"lr": 1e-2}}},
        vllm_config={"max_model_len": P + R + 8, "kv_cache_tokens": 1 << 14}))
    g = torch.Generator().manual_seed(0)
    try:
        client.call("sync_weights")
        prompts = [torch.randint(3, 200, (int(torch.randint(8, P, (1,), generator=g)),), generator=g).tolist() for _ in range(n_prompts)]
        outs = client.call("generate", prompts, {"n": n, "temperature": 1.0, "max_tokens": R, "min_p": 0.01, "seed": 1})
        B = len(outs)
        ids, mask = torch.zeros((B, P + R), dtype=torch.int64), torch.zeros((B, P + R), dtype=torch.int64)
        for i, o in enumerate(outs):
            p, t = prompts[o["prompt_index"]], o["token_ids"]
            ids[i, P - len(p):P], mask[i, P - len(p):P] = torch.tensor(p), 1
            ids[i, P:P + len(t)], mask[i, P:P + len(t)] = torch.tensor(t), 1
        batch = {"input_ids": ids, "attention_mask": mask, "response_mask": mask[:, P:].contiguous()}
        teacher = client.call("fwd_no_grad", {"batch": batch, "meta": {"top_logprobs": 32}}, reference_model=True)["batch"]
        assert teacher["top_ids"].shape == (B, R, 32)
        batch.update(teacher_top_ids=teacher["top_ids"], teacher_top_logprobs=teacher["top_log_probs"], teacher_rest=teacher["top_rest"])
        how = {"loss_fn": "distill", "loss_kwargs": {"reverse": 0.5}}
        same = client.call("fwd_bwd", {"batch": batch, "meta": {}}, how)
        assert abs(same["avg_loss"]) < 1e-2                      # the trainer still has the teacher's weights
        client.call("step")
        m = batch["response_mask"].bool()
        # a teacher that wants other tokens: its named ones moved by one
        batch["teacher_top_ids"] = torch.where(m[..., None], (teacher["top_ids"] + 1) % 32000, -1)
        out = client.call("fwd_bwd", {"batch": batch, "meta": {}}, how)
        st = client.call("step")
        assert out["avg_loss"] > 0 and st["metrics"]["grad_norm"] > 0
        assert out["metrics"]["distill/divergence"] > 0
        _lib.check_status("distillation")
    finally:
        client.call("shutdown")
