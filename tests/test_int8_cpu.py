"""8-bit products: layouts, refusals and the C entry points' checks (no GPU call is made)."""

import copy

import pytest
import torch

from multi_lora_amd import _ffi
from multi_lora_amd.kernels import Int8Rows, int8_linear, int8_matmul, quantize_rows
from multi_lora_amd.kernels.int8 import MAX_K
from multi_lora_amd.layers import Int8Linear, quantize_base


def rows(n=4, k=7):
    return Int8Rows.from_codes(torch.arange(n * k).reshape(n, k).to(torch.int8), torch.rand(n))


def test_codes_in_blocks():
    codes = torch.randint(-127, 128, (37, 130)).to(torch.int8)
    r = Int8Rows.from_codes(codes, torch.rand(37))
    assert r.codes.shape == (4, 3, 4, 16, 16) and r.shape == (37, 130)
    for row, e in ((0, 0), (36, 129), (15, 63), (16, 64), (20, 17), (5, 127), (31, 128)):
        assert r.codes[e // 64, row // 16, e // 16 % 4, row % 16, e % 16] == codes[row, e]
    assert torch.equal(r.to_rows(), codes)
    assert int((r.codes != 0).sum()) == int((codes != 0).sum())  # zeros behind columns and rows
    want = codes.double() * r.scales.double()[:, None]
    assert torch.allclose(r.dequantize().double(), want, rtol=2.0 ** -24, atol=0)


@pytest.mark.parametrize("cuts", [(0, 16, 37), (0, 5, 32, 37), (0, 0, 32, 37), (0, 37, 37)])
def test_slices_and_their_union(cuts):
    codes = torch.randint(-127, 128, (37, 100)).to(torch.int8)
    r = Int8Rows.from_codes(codes, torch.rand(37))
    parts = [r.rows(a, b) for a, b in zip(cuts, cuts[1:])]
    for p, a, b in zip(parts, cuts, cuts[1:]):
        assert torch.equal(p.to_rows(), codes[a:b]) and torch.equal(p.scales, r.scales[a:b])
        if a % 16 == 0 and b > a:
            assert p.codes.data_ptr() == r.codes[:, a // 16:].data_ptr()  # a view
    both = Int8Rows.cat(parts)
    assert torch.equal(both.to_rows(), codes) and torch.equal(both.scales, r.scales)


BAND = torch.zeros(2, 1, 4, 16, 16, dtype=torch.int8)


@pytest.mark.parametrize("make", [
    lambda: Int8Rows(torch.zeros(2, 128, dtype=torch.int8), torch.ones(2), 100),       # rows of codes
    lambda: Int8Rows(BAND[:1], torch.ones(2), 100),                                    # not padded
    lambda: Int8Rows(BAND.float(), torch.ones(2), 100),
    lambda: Int8Rows(BAND, torch.ones(17), 100),                                          # rows of another band
    lambda: Int8Rows(BAND, torch.ones(2).half(), 100),
    lambda: Int8Rows(BAND, torch.ones(2), 0),
    lambda: Int8Rows(BAND.transpose(2, 3).contiguous().transpose(2, 3), torch.ones(2), 100),
    lambda: Int8Rows(torch.zeros(2049, dtype=torch.int8)[1:].view(2, 1, 4, 16, 16), torch.ones(2), 100),  # not aligned
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
    quant = lambda x=p, xs=64, m=4, k=64, c=p, s=p, dt=bf: lib.mlora_quantize_rows(x, xs, m, k, c, s, dt, None)  # noqa: E731
    assert quant(dt=9) == -1 and quant(k=0) == -1 and quant(m=-1) == -1 and quant(xs=63) == -1
    assert quant(x=None) == -1 and quant(k=(1 << 17) + 1, xs=1 << 20) == -2 and quant(c=p + 8) == -2
    assert quant(m=0) == 0

    def mat(a=p, as_=1024, sa=p, m=4, b=p, bs=1024, sb=p, n=8, k=64, o=p, os=8, dt=bf):
        return lib.mlora_int8_matmul(a, as_, sa, m, b, bs, sb, n, k, None, o, os, dt, None)

    assert mat(dt=_ffi.MLORA_F32) == -2 and mat(n=-1) == -1 and mat(k=0) == -1 and mat(os=7) == -1
    assert mat(as_=1008) == -1 and mat(bs=1008) == -1 and mat(as_=1032) == -2 and mat(bs=1032) == -2
    assert mat(b=p + 1) == -2 and mat(a=p + 1) == -2 and mat(a=None) == -1 and mat(m=0) == 0 and mat(n=0) == 0

    def lin(x=p, xs=64, m=100, b=p, n=8, k=64, o=p, ws=p, nb=1 << 20):
        return lib.mlora_int8_linear(x, xs, m, b, 1024, p, n, k, None, o, 8, bf, ws, nb, None)

    assert lin(xs=63) == -1 and lin(x=None) == -1 and lin(ws=None) == -3 and lin(nb=100) == -3 and lin(ws=p + 4) == -2
    assert lin(m=0) == 0
    assert lib.mlora_int8_linear_workspace_bytes(100, 64) == 112 * 128 + 100 * 4
    assert lib.mlora_int8_linear_workspace_bytes(2, 4096) == 0 == lib.mlora_int8_linear_workspace_bytes(0, 64)


def test_sums_fit_32_bits():
    """The longest rows, every code -128 in both: one element more would wrap."""
    assert 128 * 128 * MAX_K < 2 ** 31 <= 128 * 128 * (MAX_K + 1)
    with pytest.raises(ValueError):
        Int8Rows.from_codes(torch.full((2, 1 << 17), -128, dtype=torch.int8), torch.ones(2))
    lib = _ffi.lib()
    p = 0x10000
    stride = (1 << 17) * 16
    assert lib.mlora_int8_matmul(p, stride, p, 1, p, stride, p, 1, 1 << 17, None, p, 1, _ffi.MLORA_BF16, None) == -2


def test_the_module_follows_its_buffers():
    """A state dict that is assigned, not copied, and a move: the weight is what the buffers hold."""
    layer, other = (Int8Linear(Int8Rows.from_codes(torch.full((20, 7), c, dtype=torch.int8), torch.full((20,), float(c)))) for c in (1, 2))
    layer.load_state_dict(other.state_dict(), assign=True)
    assert torch.equal(layer.weight.dequantize(), torch.full((20, 7), 4.0))
    assert layer.weight.codes is layer.codes
    layer = layer.bfloat16()
    assert layer.weight.scales.dtype == torch.float32 and torch.equal(layer.weight.dequantize(), torch.full((20, 7), 4.0))
    copied = copy.deepcopy(layer)
    copied.codes.zero_()
    assert not copied.weight.dequantize().any() and layer.weight.dequantize().all()


def test_a_layer_alone_is_not_a_model():
    with pytest.raises(ValueError, match="from_linear"):
        quantize_base(torch.nn.Linear(4, 4).bfloat16())
