"""A fused group after a call that raised: the next call computes, it returns nothing of the call before."""

import pytest
import torch
import torch.nn as nn

from multi_lora_amd.layers import LinearWithLoRA, fuse_qkv_projections


class Flaky:
    """A backend whose call raises once."""

    def __init__(self) -> None:
        self.calls = 0

    def apply_lora_multi(self, x, a, b, out, cols):
        self.calls += 1
        if self.calls == 2:
            raise RuntimeError("once")
        return out


def group():
    torch.manual_seed(0)
    ws = {f"m.{n}": LinearWithLoRA(nn.Linear(8, 4, bias=False)) for n in ("q_proj", "k_proj", "v_proj")}
    assert fuse_qkv_projections(ws) == 1
    return ws


@torch.no_grad()
def test_a_call_that_raised_leaves_no_answer():
    ws = group()
    backend = Flaky()
    for w in ws.values():
        w.set_lora_info(backend, torch.zeros(1, 2, 8), torch.zeros(1, 4, 2))
    first, second = torch.randn(3, 1, 8), torch.randn(3, 1, 8)
    q, k = ws["m.q_proj"], ws["m.k_proj"]
    assert torch.equal(q(first), nn.functional.linear(first, q.base_layer.weight))
    with pytest.raises(RuntimeError, match="once"):
        q(second)
    assert torch.equal(q(second), nn.functional.linear(second, q.base_layer.weight))
    assert torch.equal(k(second), nn.functional.linear(second, k.base_layer.weight))
    assert backend.calls == 3


@torch.no_grad()
def test_a_product_that_raised_leaves_no_answer():
    ws = group()
    q = ws["m.q_proj"]
    first, wrong = torch.randn(3, 1, 8), torch.randn(3, 1, 9)
    q(first)
    for _ in range(2):
        with pytest.raises(RuntimeError):
            q(wrong)
    assert torch.equal(q(first), nn.functional.linear(first, q.base_layer.weight))
