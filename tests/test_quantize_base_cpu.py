"""Which layers of a model quantize_base replaces, and what it refuses (the quantisation itself in plain torch)."""

import pytest
import torch
import torch.nn as nn
from torch.nn.utils import prune

from multi_lora_amd import Int8Linear, layers, quantize_base
from multi_lora_amd.kernels import Int8Rows
from multi_lora_amd.layers import LinearWithLoRA


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    def rows(w):
        top = w.double().abs().amax(1, keepdim=True).clamp(min=2.0 ** -100)
        return Int8Rows.from_codes(torch.round(w.double() * 127 / top).to(torch.int8), (top[:, 0] / 127).float())
    monkeypatch.setattr(layers, "quantize_rows", rows)


def linear(k=8, n=6):
    return nn.Linear(k, n, dtype=torch.bfloat16)


def test_a_layer_under_two_names_is_replaced_under_both():
    shared = linear()
    model = nn.ModuleDict(dict(a=shared, b=nn.ModuleDict(dict(c=shared, d=linear()))))
    assert quantize_base(model) == 2
    assert isinstance(model["a"], Int8Linear) and model["a"] is model["b"]["c"]
    assert isinstance(model["b"]["d"], Int8Linear)


def test_a_wrapper_under_two_names():
    wrapper = LinearWithLoRA(linear())
    model = nn.ModuleDict(dict(a=wrapper, b=wrapper))
    assert quantize_base(model) == 1 and isinstance(wrapper.base_layer, Int8Linear)


def test_a_shared_layer_stays_where_its_name_is_skipped():
    shared = linear()
    model = nn.ModuleDict(dict(a=shared, lm_head=shared))
    assert quantize_base(model) == 1
    assert isinstance(model["a"], Int8Linear) and model["lm_head"] is shared


HOOKS = {
    "forward": lambda m: m.register_forward_hook(lambda *a: None),
    "forward with arguments": lambda m: m.register_forward_hook(lambda *a: None, with_kwargs=True),
    "before": lambda m: m.register_forward_pre_hook(lambda *a: None),
    "backward": lambda m: m.register_full_backward_hook(lambda *a: None),
    "before backward": lambda m: m.register_full_backward_pre_hook(lambda *a: None),
    "state": lambda m: m.register_state_dict_post_hook(lambda *a: None),
    "before state": lambda m: m.register_state_dict_pre_hook(lambda *a: None),
    "before load": lambda m: m.register_load_state_dict_pre_hook(lambda *a: None),
    "after load": lambda m: m.register_load_state_dict_post_hook(lambda *a: None),
}


@pytest.mark.parametrize("kind", HOOKS)
def test_layers_with_hooks_are_refused_before_any_is_replaced(kind):
    """What watches a layer would be lost with it."""
    model = nn.ModuleDict(dict(a=linear(), b=linear(), lm_head=linear()))
    handle = HOOKS[kind](model["b"])
    with pytest.raises(RuntimeError, match="b has hooks"):
        quantize_base(model)
    assert type(model["a"]) is nn.Linear
    assert quantize_base(model, skip=("lm_head", "b")) == 1
    handle.remove()
    HOOKS[kind](model["lm_head"])  # (stays, and its hook with it)
    assert quantize_base(model) == 1


def test_layers_whose_weight_is_computed_are_refused():
    """torch's pruning keeps another parameter and a hook that makes the weight of it."""
    model = nn.ModuleDict(dict(a=linear()))
    prune.l1_unstructured(model["a"], "weight", 4)
    with pytest.raises(RuntimeError, match="a has hooks"):
        quantize_base(model)


def test_subclasses_stay():
    class Scaled(nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    model = nn.ModuleDict(dict(a=Scaled(8, 6, dtype=torch.bfloat16), b=linear()))
    assert quantize_base(model) == 1 and type(model["a"]) is Scaled


@pytest.mark.parametrize("training", [True, False])
def test_mode_is_kept(training):
    model = nn.ModuleDict(dict(a=linear())).train(training)
    quantize_base(model)
    assert model["a"].training == training


def test_a_wrapper_alone():
    """A model that is one wrapped layer."""
    wrapper = LinearWithLoRA(linear())
    assert quantize_base(wrapper) == 1 and isinstance(wrapper.base_layer, Int8Linear)
