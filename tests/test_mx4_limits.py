"""``ffn_format="mxfp4"``: what a configuration or a model asks for and the 4-bit layers do not do is refused before anything runs."""
import dataclasses

import pytest
import torch

from jittorinfer_b200.config import ServerConfig, load_yaml
from jittorinfer_b200.models.deepseek2 import DeepSeek2Model
from jittorinfer_b200.models.hparams import preset
from jittorinfer_b200.models.weights import random_weights


@pytest.mark.parametrize("body,fits", [("layer_split_gpus: 4\n", False), ("layer_split_gpus: 2\nsplit_mode: LLAMA_SPLIT_MODE_LAYER\n", False),
                                       ("layer_split_gpus: 1\n", True), ("layer_split_gpus: 0\n", True)])
def test_layers_on_several_gpus_are_refused(tmp_path, body, fits):
    p = tmp_path / "c.yaml"
    p.write_text("random_init: tiny\n" + body)
    plain = load_yaml(str(p))
    assert plain.split_mode == ServerConfig().split_mode == "LLAMA_SPLIT_MODE_LAYER"
    p.write_text("random_init: tiny\nffn_format: mxfp4\n" + body)
    if fits:
        load_yaml(str(p))
    else:
        with pytest.raises(ValueError, match="layer_split_gpus"):
            load_yaml(str(p))


@pytest.mark.parametrize("over", [dict(n_expert=288, n_expert_used=4), dict(n_expert=64, n_expert_used=33), dict(n_expert=80, n_group=40, topk_group=20)])
def test_more_than_the_gate_takes_is_refused_before_weights_are_read(over):
    hp = dataclasses.replace(preset("tiny-v2"), **over)

    def weights():
        raise AssertionError("a weight was read")
        yield
    with pytest.raises(ValueError, match="at most 32 of 256 in 32"):
        DeepSeek2Model(hp, weights(), dtype=torch.float32, ffn_format="mxfp4")


def test_shared_experts_beyond_the_choices_of_a_token_run_apart():
    hp = dataclasses.replace(preset("tiny-v2"), n_expert=64, n_expert_used=31, n_group=1, topk_group=1)
    assert hp.n_expert_shared == 2
    m = DeepSeek2Model(hp, random_weights(hp, seed=0, std=0.05).items(), dtype=torch.float32, ffn_format="mxfp4")
    L = next(x for x in m.layers if x.is_moe)
    assert L.shared_gu is not None and L.ffn_gu.batch == 64 and L.n_shared_merged == 0
