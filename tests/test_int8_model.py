"""Which models take ``quantization="int8"``: asked before their weights are read, and nothing is changed where the answer is no."""
import json
from dataclasses import replace

import pytest
import torch

from conftest import TINY_B, TINY_C
from nanohybrid_vlm_b200.config.registry import ARCHITECTURES
from nanohybrid_vlm_b200.engine.model import CausalLM
from nanohybrid_vlm_b200.parts.spec import LayerSpec, PartUse, part
from test_muvonex_config import CFG as OTHER


def spec_of(raw):
    import nanohybrid_vlm_b200.models  # noqa: F401
    entry = ARCHITECTURES.resolve(raw)
    return entry.build_spec(entry.parse_config(raw))


def model(raw, **last_layer):
    """``raw`` with parts of its last layer replaced."""
    spec = spec_of(raw)
    uses = {name: PartUse(last_layer.get(name, use.spec), use.prefix) for name, use in spec.layers[-1].parts}
    layer = LayerSpec(last_layer.get("block", spec.layers[-1].block), **uses)
    return CausalLM(replace(spec, layers=spec.layers[:-1] + (layer,)), torch.float32, "cpu")


def norms_of(m):
    return [p for block in m.blocks for name, p in block.parts.items() if name.endswith("norm")]


@pytest.mark.parametrize("raw", [TINY_B, TINY_C])
def test_a_model_that_has_the_form(raw):
    m = model(raw)
    kinds = [p.spec.kind for p in m.int8_parts()]
    assert kinds.count("rmsnorm") == kinds.count("gqa_attention") + kinds.count("swiglu") == 2 * len(m.blocks)
    assert not any(n.int8 for n in norms_of(m))                 # asked, not told


@pytest.mark.parametrize("other, text", [
    (dict(ffn=part("clamped_glu", intermediate_size=32, limit=7.0, alpha=1.702)), "clamped_glu"),
    (dict(mixer_norm=part("rmsnorm", width=TINY_C["hidden_size"], eps=1e-6, groups=2)), "rmsnorm"),
    (dict(ffn_norm=part("rmsnorm", width=TINY_C["hidden_size"], eps=1e-6, post_scale="gamma")), "rmsnorm"),
    (dict(ffn_norm=part("dyntanh", width=TINY_C["hidden_size"])), "dyntanh"),
    (dict(ffn=part("swiglu", intermediate_size=131080)), "131080 inputs"),
])
def test_one_layer_without_it(other, text):
    m = model(TINY_C, **other)
    for ask in (m.int8_parts, m.to_int8):
        with pytest.raises(ValueError, match=text):
            ask()
    assert not any(getattr(n, "int8", False) for n in norms_of(m))


def test_a_norm_wider_than_the_kernels_rows():
    wide = TINY_C | dict(hidden_size=51208)
    with pytest.raises(ValueError, match="rmsnorm"):
        model(wide).int8_parts()
    assert model(TINY_C | dict(hidden_size=51200)).int8_parts()


def test_refused_before_the_weights_are_read(tmp_path, monkeypatch):
    """A folder that holds a configuration and no weights: the answer does not come from the loader."""
    from nanohybrid_vlm_b200.config import Config
    from nanohybrid_vlm_b200.engine import runner
    (tmp_path / "config.json").write_text(json.dumps(OTHER))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "set_device", lambda device: None)
    monkeypatch.setattr(runner, "load_library", lambda: None)
    with pytest.raises(ValueError, match="8-bit"):
        runner.ModelRunner(Config(str(tmp_path), dtype="float32", quantization="int8", max_model_len=64, num_kvcache_blocks=4), device="cpu")
