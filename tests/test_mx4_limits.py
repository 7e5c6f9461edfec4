"""``ffn_format="mxfp4"``: what a configuration or a model asks for and the 4-bit layers do not do is refused before anything runs."""
import pytest

from jittorinfer_b200.config import ServerConfig, load_yaml


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
