"""Arguments of the 8-bit cache's operators that a kernel would take on trust: what is refused on the host, without a GPU."""
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
