"""Distillation through the pipeline on CPU: the teacher's most likely tokens from a forward pass, the student's loss and gradients from them."""
import copy
import math

import pytest
import torch

from arctic_platform_b200.engine.reference_sampler import LogitsProcessor, ReferenceSampler, shaping_of
from arctic_platform_b200.engine.sampler import SamplingParams
from arctic_platform_b200.engine.worker import EngineWorker
from arctic_platform_b200.models.decoder import top_token_logprobs, token_logprobs
from arctic_platform_b200.ops import distill
from arctic_platform_b200.rl.processors.pipeline import pack_for_model
from tests.test_zorro_equivalence_cpu import make_grpo_batch


def worker(job_type, seed, model="qwen3-tiny"):
    w = EngineWorker("cpu")
    w.initialize({"model_name": model, "job_type": job_type, "seed": seed})
    return w


def wire(seed=8, n_prompts=2, n_samples=3):
    ids, mask, R = make_grpo_batch(n_prompts=n_prompts, n_samples=n_samples, seed=seed)
    return {"input_ids": ids, "attention_mask": mask, "response_mask": mask[:, -R:].contiguous()}, R


def taught(batch, k, **meta):
    out = worker("log_prob", 5).forward_no_grad(batch, {"top_logprobs": k, **meta})["batch"]
    return {**batch, "teacher_top_ids": out["top_ids"], "teacher_top_logprobs": out["top_log_probs"], "teacher_rest": out["top_rest"]}, out


@pytest.mark.parametrize("dedup", [True, False])
def test_a_forward_pass_answers_its_most_likely_tokens(dedup):
    batch, R = wire()
    w = worker("log_prob", 2)
    meta = {"zorro_train_enable": dedup, "temperature": 0.7}
    plain = w.forward_no_grad(batch, meta)["batch"]
    asked = w.forward_no_grad(batch, {**meta, "top_logprobs": 9, "num_micro_batches": 2})["batch"]
    by_name = w.forward_no_grad(batch, meta, {"post": ["compute_top_logprobs"]})["batch"]
    assert set(asked) - set(plain) == {"top_log_probs", "top_ids", "top_rest"} and by_name["top_ids"].shape[-1] == 64
    torch.testing.assert_close(asked["log_probs"], plain["log_probs"], atol=1e-5, rtol=0)
    B = batch["input_ids"].shape[0]
    assert asked["top_log_probs"].shape == asked["top_ids"].shape == (B, R, 9) and asked["top_rest"].shape == (B, R)
    m = batch["response_mask"].bool()
    assert bool((asked["top_ids"][~m] == -1).all()) and bool((asked["top_log_probs"][~m] == 0).all())
    total = asked["top_log_probs"].exp().sum(-1) + asked["top_rest"].exp()
    torch.testing.assert_close(total[m], torch.ones(int(m.sum())), atol=1e-5, rtol=0)
    # a response token that is among the most likely has its own log-probability there
    tokens = batch["input_ids"][:, -R:]
    same = (asked["top_ids"] == tokens[..., None]) & m[..., None]
    torch.testing.assert_close(asked["top_log_probs"][same], asked["log_probs"][..., None].expand_as(same)[same], atol=1e-5, rtol=0)
    with pytest.raises(ValueError):
        w.forward_no_grad(batch, {"top_logprobs": -3})
    with pytest.raises(ValueError):
        w.forward_no_grad(batch, {"top_logprobs": 10 ** 6})


@pytest.mark.parametrize("kwargs", [{}, {"reverse": 1.0}, {"reverse": 0.4, "ce_coeff": 0.3, "entropy_coeff": 0.1, "loss_agg_mode": "seq-mean-token-mean"}])
def test_the_loss_and_its_gradients_are_the_formula(kwargs):
    batch, R = wire()
    batch["response_mask"][0, 1] = 0                              # a position without loss
    batch, _ = taught(batch, 12)
    batch["teacher_top_ids"][~batch["response_mask"].bool()] = 0     # whatever stands there
    w = worker("training", 2)
    model = copy.deepcopy(w.engine.model)
    w.engine.zero_grad()
    out = w.forward_backward(batch, {}, {"loss_fn": "distill", "loss_kwargs": kwargs})
    pk = pack_for_model(batch, {}, False)
    h = model.forward_hidden(pk.input_ids, pk.positions, pk.layout).index_select(0, pk.pred_index)
    take = lambda n: pk.gather_from_grid(batch[n])                # noqa: E731
    value, lp, ent = distill.distill_ref(h, model.output_weight, pk.labels, take("teacher_top_ids"), take("teacher_top_logprobs"), take("teacher_rest"),
                                         1.0, kwargs.get("reverse", 0.0))
    m = take("response_mask").float()
    per = value - kwargs.get("ce_coeff", 0.0) * lp - kwargs.get("entropy_coeff", 0.0) * ent
    if "loss_agg_mode" in kwargs:
        seq = pk.out_index // R
        loss = sum((per * m)[seq == s].sum() / m[seq == s].sum() for s in seq.unique()) / len(seq.unique())
    else:
        loss = (per * m).sum() / m.sum()
    assert out["avg_loss"] == pytest.approx(float(loss.detach()), rel=1e-5)
    assert out["metrics"]["distill/divergence.sum"] == pytest.approx(float((value * m).sum().detach()), rel=1e-5)
    loss.backward()
    w.engine.collect_autograd_grads()
    for (name, p), (_, q) in zip(w.engine.model.named_parameters(), model.named_parameters()):
        got = p.grad if p.grad is not None else getattr(p, "grad_f32", None)
        torch.testing.assert_close(got.float(), q.grad.float(), atol=1e-5, rtol=1e-3, msg=name)


def test_a_student_that_is_its_own_teacher_has_nothing_to_learn():
    batch, _ = wire()
    w = worker("log_prob", 5)
    batch, _ = taught(batch, 16, temperature=0.8)
    r = w.forward_no_grad(batch, {"temperature": 0.8}, {"loss_fn": "distill", "loss_kwargs": {"reverse": 0.5}})
    assert abs(r["avg_loss"]) < 1e-5 and float(r["batch"]["divergence"].abs().max()) < 1e-4
    other = worker("log_prob", 6).forward_no_grad(batch, {"temperature": 0.8}, {"loss_fn": "distill"})
    assert other["avg_loss"] > 1e-3
    # options stand in the call's own arguments or, as those of the policy losses, in the actor's
    actor, call = (worker("log_prob", 6).forward_no_grad(batch, {"temperature": 0.8, **m}, {"loss_fn": "distill", "loss_kwargs": k})["avg_loss"]
                   for m, k in (({"actor_config": {"reverse": 1.0}}, {}), ({}, {"reverse": 1.0})))
    assert actor == pytest.approx(call) and actor != pytest.approx(other["avg_loss"])


def test_micro_batches_add_up_and_refusals():
    batch, R = wire()
    batch, _ = taught(batch, 6)
    w = worker("log_prob", 2)
    one = w.forward_no_grad(batch, {}, {"loss_fn": "distill"})
    three = w.forward_no_grad(batch, {"num_micro_batches": 3}, {"loss_fn": "distill"})
    assert three["avg_loss"] == pytest.approx(one["avg_loss"], rel=1e-5)
    torch.testing.assert_close(one["batch"]["divergence"], three["batch"]["divergence"], atol=1e-5, rtol=1e-4)
    run = lambda b, **kw: w.forward_no_grad(b, {}, {"loss_fn": "distill", "loss_kwargs": kw})      # noqa: E731
    without = {k: v for k, v in batch.items() if k != "teacher_rest"}
    assert math.isfinite(run(without)["avg_loss"])
    for key in ("teacher_top_ids", "teacher_top_logprobs"):
        with pytest.raises(KeyError):
            run({k: v for k, v in batch.items() if k != key})
    with pytest.raises(ValueError):
        run({**batch, "teacher_rest": batch["teacher_rest"][:, :-1]})
    with pytest.raises(ValueError):
        run({**batch, "teacher_top_ids": batch["teacher_top_ids"][..., 0]})
    with pytest.raises(ValueError):
        run(batch, reverse=1.5)
    with pytest.raises(NotImplementedError):
        run({**batch, "action_mask_tokens": torch.zeros((len(batch["input_ids"]), R, 2), dtype=torch.int64)})


def test_rows_without_predictions():
    batch, R = wire()
    model = worker("log_prob", 2).engine.model
    pk = pack_for_model(batch, {}, False)
    lp, _ = token_logprobs(model, pk, 1.0)
    empty = top_token_logprobs(model, torch.zeros((0, model.cfg.hidden_size)), 5)
    assert lp.numel() and [tuple(t.shape) for t in empty] == [(0, 5), (0, 5), (0,)]


def test_min_p_of_sampling_params():
    assert SamplingParams.from_dict({"min_p": 0.2}).min_p == 0.2 and SamplingParams().min_p == 0.0
    assert LogitsProcessor(shaping_of(SamplingParams(min_p=0.5))).active and not LogitsProcessor(shaping_of(SamplingParams())).active
    assert shaping_of({"min_p": 0.1}) == {"min_p": 0.1} and shaping_of(None) is None
    from arctic_platform_b200.models.config import PRESETS
    s = ReferenceSampler(PRESETS["qwen3-tiny"])
    s.model.init_weights(seed=3)
    a = s.generate([[1, 2, 3]], SamplingParams(max_tokens=4, temperature=1.0, min_p=1.0, seed=1))
    b = s.generate([[1, 2, 3]], SamplingParams(max_tokens=4, temperature=0.0))
    assert a[0]["token_ids"] == b[0]["token_ids"]
