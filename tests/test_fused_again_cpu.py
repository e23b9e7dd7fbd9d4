"""A fused group's projection called again with the same tensor computes again."""

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from multi_lora_amd.layers import LinearWithLoRA, fuse_qkv_projections

LEAVES = ("q_proj", "k_proj", "v_proj")


class AddOne:
    """A backend without the multi-slice call; its delta is 1, added in place."""

    def apply_lora(self, x, a, b, base):
        return base.add_(1)


def group(seed=0):
    torch.manual_seed(seed)
    ws = {f"m.{n}": LinearWithLoRA(nn.Linear(8, 4, bias=False)) for n in LEAVES}
    assert fuse_qkv_projections(ws) == 1
    return ws


@torch.no_grad()
def test_weights_loaded_between_two_calls():
    ws, others = group(), group(1)
    x = torch.randn(3, 1, 8)
    before = [w(x).clone() for w in ws.values()]
    for w, o in zip(ws.values(), others.values()):
        w.load_state_dict(o.state_dict())
    for w, old in zip(ws.values(), before):
        assert torch.equal(w(x), F.linear(x, w.base_layer.weight)) and not torch.equal(w(x), old)


@torch.no_grad()
def test_an_input_changed_in_place():
    ws = group()
    x = torch.randn(3, 1, 8)
    for _ in range(3):
        for w in ws.values():
            assert torch.equal(w(x), F.linear(x, w.base_layer.weight))
        x.mul_(2)


@pytest.mark.parametrize("order", [(0, 1, 2, 0, 1, 2), (0, 0, 0), (2, 1, 2, 0, 0, 1)])
@torch.no_grad()
def test_a_delta_is_added_once(order):
    ws = list(group().values())
    for w in ws:
        w.set_lora_info(AddOne(), torch.zeros(1, 2, 8), torch.zeros(1, 4, 2))
    x = torch.randn(3, 1, 8)
    got = [(i, ws[i](x)) for i in order]
    for i, y in got:
        assert torch.equal(y, F.linear(x, ws[i].base_layer.weight) + 1)


@torch.no_grad()
def test_the_product_is_computed_once_for_the_three(monkeypatch):
    ws = group()
    calls = []
    real = F.linear
    monkeypatch.setattr(F, "linear", lambda *a: calls.append(1) or real(*a))
    x = torch.randn(3, 1, 8)
    for w in ws.values():
        w(x)
    assert len(calls) == 1


@torch.no_grad()
def test_an_input_changed_between_two_projections():
    ws = group()
    q, k, v = ws.values()
    x = torch.randn(3, 1, 8)
    q(x)
    x.mul_(2)
    assert torch.equal(k(x), F.linear(x, k.base_layer.weight))
    assert torch.equal(v(x), F.linear(x, v.base_layer.weight))
