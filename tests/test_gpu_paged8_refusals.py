"""Gradients that the 8-bit cache's operators would drop are refused, in the native form and in Python (GPU)."""

from types import SimpleNamespace

import pytest
import torch

from multi_lora_amd import _ffi
from multi_lora_amd.kernels import paged_attention_fp8, rotary_paged_write_fp8

from tests.test_gpu_paged8 import cache_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_pools_that_want_a_gradient(dev, monkeypatch, native):
    q, pool, table, step = cache_case(dev, [3, 1], [0, 20], 4, 2, 64, 16, torch.float16, 3)
    if not native:
        none = lambda *a: None  # noqa: E731
        monkeypatch.setattr(_ffi, "calls", lambda: SimpleNamespace(page_tables=none, paged_write8=none, paged_attention8=none))
    k, cos = torch.randn(4, 128, device=dev).half(), torch.randn(4, 64, device=dev).half()
    want = paged_attention_fp8(q, pool, step, 0.125)
    for t in (pool.keys, pool.values):
        t.requires_grad_()
        with pytest.raises(RuntimeError, match="no backward pass"):
            paged_attention_fp8(q, pool, step, 0.125)
        with pytest.raises(RuntimeError, match="no backward pass"):
            rotary_paged_write_fp8(q, k, k, cos, cos, pool, step)
        with torch.no_grad():
            assert torch.equal(paged_attention_fp8(q, pool, step, 0.125), want)
        t.requires_grad_(False)
