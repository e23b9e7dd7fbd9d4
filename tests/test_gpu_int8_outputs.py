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


@pytest.mark.parametrize("m,n", [(1, 40), (5, 33), (40, 50), (520, 4100)])
def test_scales_far_apart(dev, m, n):
    """Rows and channels whose scales lie at either end of the type's range, with products in the middle of it: no partial
    product leaves fp32.  Channels of zeros and rows of zeros stay 0."""
    k = 200
    x = activations(m, k, torch.bfloat16, 3)
    codes, scales = weight(n, k, 4)
    scales = scales / 0.01  # up to 1
    for ex, ew in ((-95, 118), (118, -95), (-60, 110), (0, 118), (118, 0)):
        xs = (x.double() * 2.0 ** ex).to(torch.bfloat16)
        ws = scales * 2.0 ** ew
        zero = codes.clone()
        zero[0] = 0
        w = Int8Rows.from_codes(zero.to(dev), ws.to(dev))
        want, slack = product(*codes_of(xs), zero, ws)
        end = want.abs() < 2.0 ** 127  # (0 and 118: some results leave the type)
        got = int8_linear(xs.to(dev), w).cpu()
        check(torch.where(end, got, 0), torch.where(end, want, 0.0), torch.where(end, slack, 0.0))
        assert not bool(torch.isnan(got).any()) and bool(end[:, 0].all())
