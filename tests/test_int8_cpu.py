"""8-bit products: layouts, refusals and the C entry points' checks (no GPU call is made)."""

import pytest
import torch

from multi_lora_amd import _ffi
from multi_lora_amd.kernels import Int8Rows, int8_linear, int8_matmul, quantize_rows


def rows(n=4, k=7):
    return Int8Rows.from_codes(torch.arange(n * k).reshape(n, k).to(torch.int8), torch.rand(n))


def test_codes_are_padded_with_zeros():
    codes = torch.randint(-127, 128, (5, 130)).to(torch.int8)
    r = Int8Rows.from_codes(codes, torch.rand(5))
    assert r.codes.shape == (5, 256) and r.shape == (5, 130)
    assert torch.equal(r.codes[:, :130], codes) and not r.codes[:, 130:].any()
    want = codes.double() * r.scales.double()[:, None]
    assert torch.allclose(r.dequantize().double(), want, rtol=2.0 ** -24, atol=0)
    both = Int8Rows.cat([r.rows(0, 2), r.rows(2, 5)])
    assert torch.equal(both.codes, r.codes) and torch.equal(both.scales, r.scales)


@pytest.mark.parametrize("make", [
    lambda: Int8Rows(torch.zeros(2, 127, dtype=torch.int8), torch.ones(2), 100),      # not padded
    lambda: Int8Rows(torch.zeros(2, 128), torch.ones(2), 100),                          # dtype
    lambda: Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(3), 100),       # scales
    lambda: Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2).half(), 100),
    lambda: Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2), 0),
    lambda: Int8Rows(torch.zeros(2, 129, dtype=torch.int8)[:, :128], torch.ones(2), 100),  # rows 129 bytes apart
    lambda: Int8Rows.from_codes(torch.zeros(2, (1 << 17) + 1, dtype=torch.int8), torch.ones(2)),
    lambda: Int8Rows.cat([rows(k=7), rows(k=8)]),
])
def test_rows_that_do_not_fit_are_refused(make):
    with pytest.raises(ValueError):
        make()


def test_there_is_no_cpu_path():
    w = rows()
    for call in (lambda: quantize_rows(torch.zeros(2, 7).bfloat16()), lambda: int8_linear(torch.zeros(2, 7).bfloat16(), w),
                 lambda: int8_matmul(w, w, torch.bfloat16)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_c_entry_points_check_before_anything_is_read():
    lib = _ffi.lib()
    bf, p = _ffi.MLORA_BF16, 1 << 20
    quant = lambda x=p, xs=64, m=4, k=64, c=p, cs=128, s=p, dt=bf: lib.mlora_quantize_rows(x, xs, m, k, c, cs, s, dt, None)  # noqa: E731
    assert quant(dt=9) == -1 and quant(k=0) == -1 and quant(m=-1) == -1 and quant(xs=63) == -1 and quant(cs=64) == -1
    assert quant(x=None) == -1 and quant(k=(1 << 17) + 1, xs=1 << 20, cs=1 << 20) == -2 and quant(c=p + 8) == -2
    assert quant(m=0) == 0

    def mat(a=p, as_=128, sa=p, m=4, b=p, bs=128, sb=p, n=8, k=64, o=p, os=8, dt=bf):
        return lib.mlora_int8_matmul(a, as_, sa, m, b, bs, sb, n, k, None, o, os, dt, None)

    assert mat(dt=_ffi.MLORA_F32) == -2 and mat(n=-1) == -1 and mat(bs=64) == -1 and mat(as_=64) == -1 and mat(os=7) == -1
    assert mat(b=p + 1) == -2 and mat(a=p + 1) == -2 and mat(a=None) == -1 and mat(m=0) == 0 and mat(n=0) == 0

    def lin(x=p, xs=64, m=100, b=p, n=8, k=64, o=p, ws=p, nb=1 << 20):
        return lib.mlora_int8_linear(x, xs, m, b, 128, p, n, k, None, o, 8, bf, ws, nb, None)

    assert lin(xs=63) == -1 and lin(x=None) == -1 and lin(ws=None) == -3 and lin(nb=100) == -3 and lin(ws=p + 4) == -2
    assert lin(m=0) == 0
    assert lib.mlora_int8_linear_workspace_bytes(100, 64) == 100 * (128 + 4)
    assert lib.mlora_int8_linear_workspace_bytes(1, 4096) == 0 == lib.mlora_int8_linear_workspace_bytes(0, 64)
