"""Products in 8-bit integers against their definitions in 64 bits."""

import pytest
import torch

from tests.int8_ref import check, codes_of, product
from multi_lora_amd.kernels import Int8Rows, int8_linear, int8_matmul, quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator("cpu").manual_seed(seed)


def activations(m, k, dtype, seed):
    """Rows as they come, with large channels; among them a row of zeros, one of one number, one whose quotients are
    often halfway between codes, and one of tiny numbers."""
    g = gen(seed)
    x = torch.randn(m, k, generator=g) * torch.where(torch.rand(k, generator=g) < 0.02, 8.0, 1.0)
    if m > 1:
        x[1] = torch.randint(-127, 128, (k,), generator=g).float()
        x[1, 0] = 254.0
    if m > 2:
        x[2] = 0
    if m > 3:
        x[3] = 0
        x[3, k // 2] = -3.0
    if m > 4:
        x[4] *= 2.0 ** -14
    return x.to(dtype)


def weight(n, k, seed):
    g = gen(seed + 1000)
    codes = torch.randint(-127, 128, (n, k), generator=g).to(torch.int8)
    return codes, torch.rand(n, generator=g) * 0.01 + 1e-4


SHAPES = [(1, 1, 1), (1, 4096, 4096), (3, 5, 7), (2, 1000, 14336), (8, 100, 4096), (8, 65, 4097), (9, 64, 256), (5, 17, 129),
          (16, 33, 130), (17, 48, 128), (32, 100, 500), (33, 64, 1024), (64, 1000, 1000), (64, 31, 4096), (65, 63, 128),
          (130, 257, 1025), (200, 4096, 256), (333, 777, 1111), (1029, 4100, 130), (2050, 2048, 256), (4000, 4100, 390)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_against_64_bits(m, n, k, dtype):
    x = activations(m, k, dtype, m + n + k)
    codes, scales = weight(n, k, m * n)
    bias = torch.randn(n, generator=gen(3)).to(dtype) if (m + n) % 2 else None
    w = Int8Rows.from_codes(codes.to(DEV), scales.to(DEV))
    got = int8_linear(x.to(DEV), w, bias.to(DEV) if bias is not None else None)
    check(got, *product(*codes_of(x), codes, scales, bias))
    # The same through rows quantised before: the same bits.
    rows = quantize_rows(x.to(DEV))
    again = int8_matmul(rows, w, dtype, bias.to(DEV) if bias is not None else None)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (7, 100), (5, 1024), (6, 1032), (9, 4096), (5, 8200), (5, 20001), (300, 512)])
def test_codes_are_those_of_exact_arithmetic(m, k, dtype):
    x = activations(m, k, dtype, m * k)
    rows = quantize_rows(x.to(DEV))
    codes, scales = codes_of(x)
    assert torch.equal(rows.to_rows().cpu().double(), codes)
    tail = rows.codes.permute(1, 3, 0, 2, 4).reshape(-1, rows.codes.shape[0] * 64)[:m, k:]
    assert not tail.any()  # zeros behind column k
    torch.testing.assert_close(rows.scales.cpu().double(), scales, rtol=2.0 ** -24, atol=0)


def test_every_quotient_of_a_type_is_rounded_as_exactly():
    """All finite bf16 numbers up to each of several maxima, ties among them."""
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    every = every[torch.isfinite(every)]
    tops = torch.tensor([1.0, 127.0, 254.0, 1.9921875, 63.5, 3.0e38, 1e-30, 100.5], dtype=torch.bfloat16)
    for top in tops:
        x = every[every.abs() <= top][None]
        rows = quantize_rows(x.to(DEV))
        assert torch.equal(rows.to_rows().cpu().double(), codes_of(x)[0]), float(top)


def test_float32_weights():
    w = torch.randn(100, 777, generator=gen(1))
    rows = quantize_rows(w.to(DEV))
    codes, scales = codes_of(w)
    # fp32 quotients next to halfway may round the other way: by one code, and the number is then next to the border.
    off = (rows.to_rows().cpu().double() - codes).abs()
    assert off.max() <= 1 and off.mean() < 1e-4
    near = (w.double() / scales[:, None] - codes).abs()[off > 0]
    assert bool((near > 0.5 - 1e-4).all())
    torch.testing.assert_close(rows.scales.cpu().double(), scales, rtol=2.0 ** -24, atol=0)


@pytest.mark.parametrize("m", [4, 100])
def test_rows_that_are_not_finite(m):
    x = activations(m, 300, torch.bfloat16, 5)
    x[0, 7], x[2, 299], x[3, 0] = float("inf"), float("nan"), float("-inf")
    codes, scales = weight(70, 300, 5)
    got = int8_linear(x.to(DEV), Int8Rows.from_codes(codes.to(DEV), scales.to(DEV)))
    check(got, *product(*codes_of(x), codes, scales))
    assert bool(torch.isnan(got[[0, 2, 3]]).all()) and bool(torch.isfinite(got[1]).all())


@pytest.mark.parametrize("m", [3, 40, 90])
def test_slices_of_wider_tensors(m):
    k, n = 200, 50
    wide = activations(m, 3 * k + 1, torch.float16, m)
    codes, scales = weight(3 * n, k, m)
    whole = Int8Rows.from_codes(codes.to(DEV), scales.to(DEV))
    w = whole.rows(n, 2 * n)
    view = whole.rows(48, 48 + n)  # blocks further apart than they are long
    assert view.codes.data_ptr() != w.codes.data_ptr() and not view.codes.is_contiguous()
    check(int8_linear(wide.to(DEV)[:, :k], view), *product(*codes_of(wide[:, :k]), codes[48:48 + n], scales[48:48 + n]))
    bias = torch.randn(n, generator=gen(2)).half()
    for at in (0, 1, k):
        x = wide.to(DEV)[:, at:at + k]
        buf = torch.full((m, 2 * n + 3), 7.0, dtype=torch.float16, device=DEV)
        for col in (0, 3):
            out = buf[:, col:col + n]
            assert int8_linear(x, w, bias.to(DEV), out=out) is out
            check(out, *product(*codes_of(wide[:, at:at + k]), codes[n:2 * n], scales[n:2 * n], bias))
        assert bool((buf[:, n + 3:] == 7).all())


def test_empty_calls():
    w = Int8Rows.from_codes(*(t.to(DEV) for t in weight(9, 33, 1)))
    assert int8_linear(torch.zeros(0, 33, dtype=torch.bfloat16, device=DEV), w).shape == (0, 9)
    assert int8_linear(torch.zeros(5, 33, dtype=torch.bfloat16, device=DEV), w.rows(3, 3)).shape == (5, 0)
    assert quantize_rows(torch.zeros(0, 33, dtype=torch.bfloat16, device=DEV)).shape == (0, 33)


def test_refusals():
    w = Int8Rows.from_codes(*(t.to(DEV) for t in weight(9, 33, 1)))
    x = torch.zeros(4, 33, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="33"):
        int8_linear(x[:, :32], w)
    with pytest.raises(ValueError):
        int8_linear(x.float(), w)
    with pytest.raises(ValueError):
        int8_linear(x.t(), w)
    with pytest.raises(ValueError, match="bias"):
        int8_linear(x, w, torch.zeros(9, device=DEV))
    with pytest.raises(ValueError, match="out"):
        int8_linear(x, w, out=torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(RuntimeError, match="backward"):
        int8_linear(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: int8_linear(t, w), x)
    with pytest.raises(RuntimeError):
        int8_linear(x.cpu(), w)
    square = Int8Rows.from_codes(*(t.to(DEV) for t in weight(33, 33, 1)))
    with pytest.raises(ValueError, match="overlaps"):
        int8_linear(x, square, out=x)
    both = torch.zeros(4, 42, dtype=torch.bfloat16, device=DEV)
    assert int8_linear(both[:, :33], w, out=both[:, 33:]).shape == (4, 9)  # side by side in one buffer
    with pytest.raises(ValueError):
        int8_matmul(w, square.rows(0, 9), torch.float32)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_captured_and_replayed(m):
    k, n = 512, 640
    codes, scales = weight(n, k, m)
    w = Int8Rows.from_codes(codes.to(DEV), scales.to(DEV))
    x = activations(m, k, torch.bfloat16, 1).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        int8_linear(x, w)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = int8_linear(x, w)
    for seed in range(2, 6):
        new = activations(m, k, torch.bfloat16, seed)
        x.copy_(new)
        eager = int8_linear(x, w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        check(out, *product(*codes_of(new), codes, scales))


def test_two_streams_at_once():
    k, n = 1024, 2048
    w = Int8Rows.from_codes(*(t.to(DEV) for t in weight(n, k, 7)))
    xs = [activations(m, k, torch.bfloat16, m).to(DEV) for m in (100, 200)]
    want = [int8_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(int8_linear(xs[i], w))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.parametrize("m,k", [(399, 130), (400, 4096), (517, 4097), (1090, 300), (701, 9000), (1025, 1024)])
def test_codes_of_many_rows(m, k):
    x = activations(m, k, torch.bfloat16, m * k)
    rows = quantize_rows(x.to(DEV))
    codes, scales = codes_of(x)
    assert torch.equal(rows.to_rows().cpu().double(), codes)
    torch.testing.assert_close(rows.scales.cpu().double(), scales, rtol=2.0 ** -24, atol=0)
    # Numbers with few bits: fp32 quotients are then those of the 16-bit type.
    again = quantize_rows(x.float().to(DEV))
    assert torch.equal(again.codes[:, :m // 16], rows.codes[:, :m // 16]) and torch.equal(again.scales, rows.scales)


@pytest.mark.parametrize("m", [1, 20, 600])
def test_the_longest_sums(m):
    """Codes of -128 throughout: the sum is the largest that 32 bits hold but 16383."""
    k, n = (1 << 17) - 1, 4100 if m == 600 else 5
    a = Int8Rows.from_codes(torch.full((m, k), -128, dtype=torch.int8, device=DEV), torch.full((m,), 2.0 ** -31, device=DEV))
    b = Int8Rows.from_codes(torch.full((n, k), -128, dtype=torch.int8, device=DEV), torch.ones(n, device=DEV))
    assert torch.equal(int8_matmul(a, b, torch.float16), torch.ones(m, n, dtype=torch.float16, device=DEV))
