"""Gradients and tangents that products in 8-bit integers would drop are refused, in the native form and in Python (GPU)."""

from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from multi_lora_amd import _ffi
from multi_lora_amd.kernels import Int8Rows, int8_linear, int8_matmul

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("m", [1, 40])
def test_scales_that_want_a_gradient(dev, monkeypatch, m, native):
    if not native:
        monkeypatch.setattr(_ffi, "calls", lambda: SimpleNamespace(int8_linear=lambda *a: None))
    g = torch.Generator().manual_seed(m)
    codes, x = torch.randint(-127, 128, (24, 100), generator=g).to(torch.int8).to(dev), torch.randn(m, 100, generator=g).bfloat16().to(dev)
    scales = torch.rand(24, generator=g).to(dev)
    plain = Int8Rows.from_codes(codes, scales)
    want = int8_linear(x, plain)
    learned = Int8Rows.from_codes(codes, scales.clone().requires_grad_())
    calls = (lambda w: int8_linear(x, w), lambda w: int8_matmul(w, plain, torch.bfloat16), lambda w: int8_matmul(plain, w, torch.bfloat16))
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward pass"):
            call(learned)
    with torch.no_grad():
        assert torch.equal(int8_linear(x, learned), want)
    with forward_ad.dual_level():
        dual = Int8Rows(plain.codes, forward_ad.make_dual(scales, torch.ones_like(scales)), 100)
        for call in calls:
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(dual)
