"""The host side of generation: drawing ids (torch refuses a bad probability on the CPU; on a GPU it would end
the process's context), and models that no step can be recorded for."""
import math
from types import SimpleNamespace

import pytest
import torch

from zs_b200 import ZsError
from zs_b200.generate import sample


@pytest.mark.parametrize("temperature", [1e-46, 1e-40, 1e-20, 1e-3])
def test_small_temperatures_draw_the_largest(temperature):
    logits = torch.tensor([[1.0, 40.0, -3.0, 39.0], [1e30, 2.0, -1e30, 0.0], [-5.0, -math.inf, -4.0, -math.inf]])
    for dtype in (torch.float32, torch.bfloat16):
        assert sample(logits.to(dtype), temperature, torch.Generator().manual_seed(0)).tolist() == [1, 0, 2]


def test_large_temperatures_draw_any_visible_id():
    logits = torch.tensor([[1.0, -math.inf, 3e38, -3e38]]).expand(20000, 4)   # shares of e^0, 0, e^3, e^-3 or more
    for temperature in (1e38, math.inf):
        got = sample(logits, temperature, torch.Generator().manual_seed(0))
        assert set(got.tolist()) == {0, 2, 3}


def test_a_draw_follows_the_softmax():
    logits = torch.log(torch.tensor([[0.5, 0.25, 0.25 - 1e-7, 1e-7]])).expand(20000, 4) * 0.7 + 3
    got = torch.bincount(sample(logits, 0.7, torch.Generator().manual_seed(1)), minlength=4) / 20000
    # four standard deviations of a share of 20000 draws
    assert (got - torch.tensor([0.5, 0.25, 0.25, 0.0])).abs().max() < 4 * 0.5 / math.sqrt(20000)


@pytest.mark.parametrize("row", [[math.nan, 1.0, 2.0], [math.inf, 1.0, math.inf], [-math.inf] * 3])
def test_rows_without_a_largest_logit_get_some_id(row):
    logits = torch.tensor([row, [0.0, 100.0, 0.0]])
    got = sample(logits, 1.0, torch.Generator().manual_seed(0)).tolist()
    assert 0 <= got[0] < 3 and got[1] == 1


def test_a_temperature_that_is_no_number_is_refused():
    with pytest.raises(ZsError, match="temperature"):
        sample(torch.zeros(1, 4), math.nan)


def test_sharded_experts_are_refused(tmp_path):
    import torch.distributed as dist

    from modeling.model_config import ModelConfig
    from scattermoe.expert_parallel import shard_experts
    from zs_b200.generate import DecodeStep, generate
    from zs_b200.lm import MoELM

    cfg = ModelConfig(vocab_size=64, embed_size=128, hidden_size=128, transformer_depth=1, intermediate_size=64,
                      n_experts=5, n_shared_experts=1, n_attention_heads=2, n_key_value_heads=1,
                      attention_window_pattern=(None,), max_position_embeddings=64, sequence_length=64)
    m = MoELM(cfg)
    cache = SimpleNamespace(kv=torch.zeros(1), seq_lens=torch.zeros(2, dtype=torch.int32))
    step = DecodeStep(m, cache)
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/group", rank=0, world_size=1)
    try:
        assert shard_experts(m)
        with pytest.raises(ZsError, match="sharded"):
            DecodeStep(m, cache)
        with pytest.raises(ZsError, match="sharded"):
            step()                                           # sharded after the step was made
        with pytest.raises(ZsError, match="sharded"):
            generate(m, [[1, 2]], 4)
        none = torch.zeros(2, dtype=torch.int32)
        with pytest.raises(ZsError, match="every rank"):     # the other ranks would wait for this one
            m.forward_paged(torch.zeros(0, dtype=torch.long), cache, none.view(1, 2), none[:1], none)
    finally:
        dist.destroy_process_group()
