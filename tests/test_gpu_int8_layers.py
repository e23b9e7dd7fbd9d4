"""8-bit projections as a model has them (GPU)."""

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from multi_lora_amd.kernels import int8_linear
from multi_lora_amd.layers import Int8Linear, fuse_gate_up_projections, fuse_qkv_projections

from tests.int8_ref import check, codes_of, product
from tests.test_int8_layers_cpu import states, wrappers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 5, 70, 700])
@pytest.mark.parametrize("widths", [(20, 24, 8), (37, 37), (160, 1, 33)])
@torch.inference_mode()
def test_groups_of_odd_widths(dev, widths, rows):
    """A fused group's columns are its layers' results, bit for bit, also after a state dict has been loaded."""
    k = 200
    ws = {n: w.to(dev) for n, w in wrappers(widths, k, 0).items()}
    (fuse_qkv_projections if len(widths) == 3 else fuse_gate_up_projections)(ws, all_shapes=True)
    x = torch.randn(rows, 1, k, generator=torch.Generator().manual_seed(rows)).bfloat16().to(dev)
    for seed in (0, 50):
        for n, state in states(wrappers(widths, k, seed)).items():
            ws[n].load_state_dict(state)
        x = x + 1
        for n, w in ws.items():
            got = w(x)
            assert got.shape == (rows, 1, w.base_layer.out_features) and torch.equal(got, w.base_layer(x))
            want = w.base_layer.weight
            check(got[:, 0], *product(*codes_of(x[:, 0]), want.to_rows().cpu(), want.scales.cpu()))


@torch.inference_mode()
def test_groups_whose_layers_are_moved_or_replaced(dev):
    k, widths = 96, (48, 20, 16)
    ws = wrappers(widths, k, 0)
    fuse_qkv_projections(ws)  # on the CPU
    for w in ws.values():
        w.to(dev)
    x = torch.randn(6, 1, k, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    for seed in (None, 50):
        if seed is not None:
            ws["layer.v_proj"].load_state_dict(wrappers(widths, k, seed)["layer.v_proj"].to(dev).state_dict(), assign=True)
        x = x * 2
        for w in ws.values():
            assert torch.equal(w(x), w.base_layer(x))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("given", [torch.float32, torch.bfloat16, torch.float16])
@torch.no_grad()
def test_under_autocast(dev, given, dtype):
    """Inputs and biases are cast to the region's type, as those of nn.Linear are; outside of one float32 is refused."""
    torch.manual_seed(3)
    layer = Int8Linear.from_linear(nn.Linear(72, 40, device=dev, dtype=torch.bfloat16))
    x = torch.randn(3, 5, 72, device=dev).to(given)
    want = int8_linear(x.to(dtype).view(15, 72), layer.weight, layer.bias.to(dtype)).view(3, 5, 40)
    with torch.autocast("cuda", dtype=dtype):
        got = layer(x)
        assert F.linear(x, torch.zeros(1, 72, device=dev)).dtype == got.dtype == dtype and torch.equal(got, want)
        with torch.autocast("cuda", enabled=False):
            if given == torch.bfloat16:
                assert layer(x).dtype == given
            else:
                with pytest.raises(ValueError):
                    layer(x)
    ws = {n: w.to(dev) for n, w in wrappers((48, 20, 16), 72, 0).items()}
    fuse_qkv_projections(ws, all_shapes=True)
    with torch.autocast("cuda", dtype=dtype):
        for w in ws.values():
            assert torch.equal(w(x), int8_linear(x.to(dtype).view(15, 72), w.base_layer.weight).view(3, 5, -1))


@pytest.mark.parametrize("given", [torch.int64, torch.float64])
@torch.no_grad()
def test_autocast_casts_no_others(dev, given):
    """As with nn.Linear: numbers of 64 bits and whole numbers are not cast, and so not taken."""
    layer = Int8Linear.from_linear(nn.Linear(72, 40, device=dev, dtype=torch.bfloat16))
    with torch.autocast("cuda", dtype=torch.bfloat16), pytest.raises(ValueError):
        layer(torch.ones(2, 72, device=dev, dtype=given))
