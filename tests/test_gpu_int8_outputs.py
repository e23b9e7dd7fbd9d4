"""Where products in 8-bit integers store their results (GPU): columns of wider tensors that begin at any element."""

import pytest
import torch

from multi_lora_amd.kernels import Int8Rows, int8_linear

from tests.int8_ref import check, codes_of, product
from tests.test_gpu_int8 import activations, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n", [(520, 4100), (520, 4096), (1100, 4101), (40, 100), (3, 68)])
def test_columns_of_wider_tensors(dev, m, n, dtype):
    """Tiles store 16 bytes at once where rows begin at multiples of them, 8 where at multiples of 8, else elements."""
    k = 130
    x = activations(m, k, dtype, m + n)
    codes, scales = weight(n, k, n)
    want = product(*codes_of(x), codes, scales)
    w, x = Int8Rows.from_codes(codes.to(dev), scales.to(dev)), x.to(dev)
    first = int8_linear(x, w)
    check(first, *want)
    for width in (n + 16, n + 12 - n % 4, n + 13):
        for col in (0, 1, 2, 4, 8):
            buf = torch.full((m, width), 7.0, dtype=dtype, device=dev)
            int8_linear(x, w, out=buf[:, col:col + n])
            assert torch.equal(buf[:, col:col + n], first)
            assert bool((buf[:, :col] == 7).all()) and bool((buf[:, col + n:] == 7).all())
