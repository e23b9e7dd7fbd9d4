"""Which layers of a model quantize_base replaces, and what it refuses (the quantisation itself in plain torch)."""

import pytest
import torch
import torch.nn as nn

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
