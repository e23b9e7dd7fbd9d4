"""8-bit projections in fused groups and in models: what the layers hold (no GPU call is made)."""

import pytest
import torch
import torch.nn as nn

from multi_lora_amd.kernels import Int8Rows
from multi_lora_amd.layers import Int8Linear, LinearWithLoRA, fuse_gate_up_projections, fuse_qkv_projections

NAMES = ("q_proj", "k_proj", "v_proj")


def rows(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    return Int8Rows.from_codes(torch.randint(-127, 128, (n, k), generator=g).to(torch.int8), torch.rand(n, generator=g))


def wrappers(widths, k, seed):
    names = NAMES if len(widths) == 3 else ("gate_proj", "up_proj")
    return {f"layer.{name}": LinearWithLoRA(Int8Linear(rows(n, k, seed + i))) for i, (name, n) in enumerate(zip(names, widths))}


def fused(widths, k, seed):
    ws = wrappers(widths, k, seed)
    assert (fuse_qkv_projections if len(widths) == 3 else fuse_gate_up_projections)(ws) == 1
    return ws


def states(ws):
    return {n: {key: t.clone() for key, t in w.state_dict().items()} for n, w in ws.items()}


def check(ws, widths, k, seed):
    """Layers and group hold the rows of ``seed``."""
    for i, (w, n) in enumerate(zip(ws.values(), widths)):
        want = rows(n, k, seed + i)
        start, end = w.qkv_slice
        assert end - start == n
        group = w.qkv_group.weight
        for got_codes, got_scales in ((w.base_layer.weight.to_rows(), w.base_layer.weight.scales),
                                      (group.to_rows()[start:end], group.scales[start:end])):
            assert torch.equal(got_codes, want.to_rows()) and torch.equal(got_scales, want.scales), f"projection {i}"


@pytest.mark.parametrize("widths", [(32, 16, 48), (20, 24, 8), (5, 1, 33), (16, 20, 20), (37, 37), (64, 20)])
def test_a_fused_group_holds_what_its_layers_load(widths):
    """State dicts saved before fusing and after it, of widths that do and do not fill bands of 16 rows; what saved codes
    hold behind their last row may be anything."""
    k = 100
    before = states(wrappers(widths, k, 50))
    for state in before.values():
        codes = state["base_layer.codes"]
        n = state["base_layer.scales"].shape[0]
        codes.permute(1, 3, 0, 2, 4)[-1, (n - 1) % 16 + 1:] = 99  # rows that do not exist
    ws = fused(widths, k, 0)
    check(ws, widths, k, 0)
    for n, w in ws.items():
        w.load_state_dict(before[n])
    check(ws, widths, k, 50)
    after = states(ws)
    again = fused(widths, k, 7)
    for n, w in again.items():
        w.load_state_dict(after[n])
    check(again, widths, k, 50)
    assert sum(w.base_layer.codes.untyped_storage().data_ptr() == w.qkv_group.weight.codes.untyped_storage().data_ptr()
               for w in again.values()) == len(widths)  # no second copy of a weight


@pytest.mark.parametrize("widths", [(32, 16, 48), (20, 24, 8)])
def test_a_fused_group_follows_buffers_that_are_replaced(widths):
    """A state dict that is assigned, not copied, and layers that are given other weights: one of them, then all."""
    k = 70
    ws = fused(widths, k, 0)
    x = torch.zeros(1, 1, k)
    one = wrappers(widths, k, 50)["layer.k_proj"]
    ws["layer.k_proj"].load_state_dict(one.state_dict(), assign=True)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ws["layer.q_proj"](x)  # (the fused product's weight is looked at before the refusal)
    group = ws["layer.q_proj"].qkv_group
    for i, (w, n) in enumerate(zip(ws.values(), widths)):
        want = rows(n, k, i + (50 if i == 1 else 0))
        start, end = w.qkv_slice
        assert torch.equal(group.weight.to_rows()[start:end], want.to_rows()), f"projection {i}"
        assert torch.equal(group.weight.scales[start:end], want.scales) and torch.equal(w.base_layer.weight.to_rows(), want.to_rows())
    for i, (w, n) in enumerate(zip(ws.values(), widths)):
        w.base_layer.weight = rows(n, k, 90 + i)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ws["layer.q_proj"](x)
    check(ws, widths, k, 90)


def test_a_layer_of_a_group_that_is_replaced():
    """By another 8-bit layer: the group has its weight.  By a 16-bit one: the group cannot be computed as one."""
    widths, k = (32, 16, 48), 70
    ws = fused(widths, k, 0)
    x = torch.zeros(1, 1, k)
    ws["layer.k_proj"].base_layer = Int8Linear(rows(16, k, 77))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ws["layer.q_proj"](x)
    assert torch.equal(ws["layer.q_proj"].qkv_group.weight.to_rows()[32:48], rows(16, k, 77).to_rows())
    ws["layer.v_proj"].base_layer = nn.Linear(k, 48, bias=False)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="8-bit and 16-bit"):
            ws["layer.q_proj"](x)
    ws["layer.v_proj"].base_layer = Int8Linear(rows(48, k, 3), torch.zeros(48))
    with pytest.raises(RuntimeError, match="bias"):
        ws["layer.q_proj"](x)
    torch.manual_seed(0)
    for w, n in zip(ws.values(), widths):  # all of them: a 16-bit group
        w.base_layer = nn.Linear(k, n, bias=False)
    x = torch.randn(2, 1, k)
    for w in ws.values():
        assert torch.allclose(w(x), w.base_layer(x), atol=1e-6)
