"""Which share of a model 8-bit weights change, and that a model of which they change nothing is refused."""
import importlib
from types import SimpleNamespace as NS

import pytest
import torch


def test_the_share_in_8_bits():
    from helpers import tiny_config, tiny_config_dict
    from tinyserve_b200.parts.model import build_model
    from tinyserve_b200.weights import check_weight_dtype
    c = tiny_config_dict("B")
    attention = c["head_dim"] * (2 * c["num_attention_heads"] + 2 * c["num_key_value_heads"]) * c["hidden_size"]
    layer = attention + 3 * c["hidden_size"] * c["intermediate_size"]
    norms = 2 * c["hidden_size"] + 2 * c["head_dim"]
    total = c["num_hidden_layers"] * (layer + norms) + 2 * c["vocab_size"] * c["hidden_size"] + c["hidden_size"]
    model = build_model(tiny_config("B"))
    assert check_weight_dtype(model, "int8") == pytest.approx(c["num_hidden_layers"] * layer / total)
    assert check_weight_dtype(model, "auto") == 0.0


@pytest.mark.parametrize("name", ["babadra", "delilorn", "dudatar", "gunulorn", "ronolorn", "tarivik"])
def test_every_architecture_has_some(name):
    from tinyserve_b200.parts.model import build_model
    from tinyserve_b200.weights import check_weight_dtype
    module = importlib.import_module(f"{name}_configs")
    for which in getattr(module, f"{name.upper()}_TINY"):
        assert 0.1 < check_weight_dtype(build_model(getattr(module, f"{name}_config")(which)), "int8") < 0.7


def test_a_model_without_any_is_refused(tmp_path):
    from tinyserve_b200.parts.base import ParamSpec
    from tinyserve_b200.weights import fill_random_on_device, load_weights
    part = NS(path="", param_specs=lambda: {"experts.weight": ParamSpec((4, 4))}, bind=lambda tensors: None)
    model = NS(named_parts=lambda: [part])
    fill_random_on_device(model, torch.float32, "cpu")
    for make in (lambda: fill_random_on_device(model, torch.float32, "cpu", 0, "int8"), lambda: load_weights(model, str(tmp_path), torch.float32, "cpu", "int8")):
        with pytest.raises(ValueError, match="no matrix of the model can be held in 8 bits"):
            make()


def test_weights_are_complete_before_the_first_product(tmp_path, monkeypatch):
    """Both ways of filling a model end with a synchronisation of its device: products over constant weights do not wait for who made them."""
    from helpers import make_model_dir, tiny_config
    from tinyserve_b200.parts.model import build_model
    from tinyserve_b200.weights import fill_random_on_device, load_weights, loader, random_init
    seen = []
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: seen.append(("device", str(device))))
    loader.settle("cuda:0")
    loader.settle(torch.device("cpu"))
    assert seen == [("device", "cuda:0")]
    bound = []
    for module in (loader, random_init):
        monkeypatch.setattr(module, "settle", lambda device: seen.append(("settled", len(bound))))
    model = build_model(tiny_config("A"))
    for part in model.named_parts():
        monkeypatch.setattr(part, "bind", lambda tensors, part=part: bound.append(part))
    n = sum(1 for _ in model.named_parts())
    fill_random_on_device(model, torch.float32, "cpu")
    load_weights(model, make_model_dir(tmp_path, "A"), torch.float32, "cpu")
    assert seen[1:] == [("settled", n), ("settled", 2 * n)]
