"""The 8-bit paged cache: layouts, refusals and the C entry points' checks (no GPU call is made)."""

import ctypes

import pytest
import torch

from multi_lora_amd import _ffi
from multi_lora_amd.decoder import DecoderConfig, PagedKV
from multi_lora_amd.kernels import Fp8Pool, PagedStep, PageState, paged_attention_fp8, rotary_paged_write_fp8

from tests import fp8_ref

CPU = torch.device("cpu")


def pool(pages=4, g=2, page=16, d=64, dtype=torch.bfloat16):
    return Fp8Pool.new(pages, g, page, d, dtype, CPU)


def test_the_reference_codes_are_torchs():
    every = torch.arange(256, dtype=torch.uint8)
    want = every.view(torch.float8_e4m3fn).double()
    got = fp8_ref.decode(every)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))
    x = torch.cat((torch.randn(2000, generator=torch.Generator().manual_seed(1)) * 100, want[~torch.isnan(want)].float()))
    x = x.clamp(-448, 448)
    assert torch.equal(fp8_ref.encode(x.double()), x.to(torch.float8_e4m3fn).view(torch.uint8))


def test_dequantised_pools():
    p = pool(page=32)
    g = torch.Generator().manual_seed(1)
    p.keys.view(torch.uint8).copy_(torch.randint(0, 127, p.keys.shape, generator=g))
    p.values.view(torch.uint8).copy_(torch.randint(0, 127, p.values.shape, generator=g))
    p.key_scales.copy_(torch.randint(100, 140, p.key_scales.shape, generator=g))
    p.value_scales.copy_(torch.randint(100, 140, p.value_scales.shape, generator=g))
    k, v = p.dequantize()
    for pg, h, at, e in ((0, 0, 0, 0), (3, 1, 31, 63), (2, 0, 15, 7), (1, 1, 16, 8)):
        for got, codes, scales, i in ((k, p.keys, p.key_scales, (pg, h, at, e)), (v, p.values, p.value_scales, (pg, h, e, at))):
            want = float(fp8_ref.decode(codes.view(torch.uint8)[i])) * 2.0 ** (int(scales[pg, h, at // 16]) - 127)
            assert float(got[i]) == want
    kv = PagedKV(DecoderConfig(), 2, 40, CPU, torch.float16, fp8=True)
    assert len(kv.pools) == 2 and kv.pools[0].shape == (6, 2, 16, 64) and kv.pools[1].dtype == torch.float16
    assert PagedKV(DecoderConfig(), 2, 40, CPU, torch.float16).pools is None


@pytest.mark.parametrize("make", [
    lambda: pool(page=8), lambda: pool(page=48), lambda: pool(page=2048), lambda: pool(d=96), lambda: pool(pages=0),
    lambda: pool(dtype=torch.float32),
    lambda: Fp8Pool(pool().keys.view(torch.uint8), pool().values.view(torch.uint8), pool().key_scales, pool().value_scales, torch.float16),
    lambda: Fp8Pool(pool().keys, pool().keys, pool().key_scales, pool().value_scales, torch.float16),
    lambda: Fp8Pool(pool().keys, pool().values, pool().key_scales[:3], pool().value_scales, torch.float16),
    lambda: Fp8Pool(pool().keys, pool().values, pool().key_scales, pool().value_scales.float(), torch.float16),
    lambda: Fp8Pool(pool(g=4).keys[:, :2].transpose(0, 1), pool().values, pool().key_scales, pool().value_scales, torch.float16),
    lambda: Fp8Pool(torch.zeros(4 * 2056, dtype=torch.uint8).view(torch.float8_e4m3fn).as_strided((4, 2, 16, 64), (2056, 1024, 64, 1)),
                    pool().values, pool().key_scales, pool().value_scales, torch.float16),  # pages 2056 bytes apart
])
def test_pools_that_do_not_fit_are_refused(make):
    with pytest.raises(ValueError):
        make()


def test_there_is_no_cpu_path():
    p = pool()
    step = PagedStep(PageState.new(2, 32, 4, 16, CPU), 2, 1)
    step.filled = True
    x = torch.zeros(2, 128).bfloat16()
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        rotary_paged_write_fp8(x, x, x, x[:, :64], x[:, :64], p, step)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        paged_attention_fp8(x, p, step, 0.1)


def test_c_entry_points_check_before_anything_is_read():
    lib = _ffi.lib()
    bf, p = _ffi.MLORA_BF16, 1 << 20

    def write(heads=4, g=2, d=64, keys=p, ks=2048, vs=2048, kscale=p, pages=4, page=16, rows=2, dt=bf):
        return lib.mlora_rotary_paged_write_fp8(p, heads * d, p, g * d, p, g * d, p, p, d, dt, p, rows, heads, g, d, keys, ks, p,
                                                vs, kscale, p, pages, page, p, heads * d, dt, None)

    assert write(page=8) == -2 and b"16 positions" in lib.mlora_last_error()
    assert write(dt=_ffi.MLORA_F32) == -2 and write(d=96) == -2 and write(ks=2000) == -1 and write(kscale=None) == -1
    assert write(keys=p + 8) == -2 and write(ks=2056) == -2 and write(rows=0) == 0

    pages = _ffi.Pages(p, 2, p, p, p, 2, 2, 4, 16)
    step = _ffi.PagedStep(p, p, p, p, p, p, 1 << 20, 1 << 24, 2, 1)

    def attend(q=p, ks=2048, scales=p, pages=pages, d=64, dt=bf):
        return lib.mlora_paged_attention_fp8(q, 256, p, ks, p, 2048, scales, p, ctypes.byref(pages), ctypes.byref(step), p, 256, 4,
                                             2, d, 0.1, dt, None)

    assert attend(pages=_ffi.Pages(p, 2, p, p, p, 2, 2, 4, 8)) == -2 and b"16 positions" in lib.mlora_last_error()
    assert attend(dt=_ffi.MLORA_F32) == -2 and attend(ks=2000) == -1 and attend(scales=None) == -1 and attend(ks=2056) == -2
    assert attend(q=p + 2) == -2
