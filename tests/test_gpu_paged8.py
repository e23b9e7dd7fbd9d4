"""The paged KV cache in 8 bits (GPU) against plain 64-bit forms, at the sizes, values and masks where it can go wrong."""

import random
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from multi_lora_amd import _ffi
from multi_lora_amd.kernels import Fp8Pool, PagedStep, PageState, page_tables, paged_attention_fp8, rotary_paged_write_fp8

from tests import fp8_ref
from tests import paged_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def bits(t):
    return t.view(torch.uint8).cpu()


def parts(pool):
    """Codes and exponents on the CPU, as the reference takes them."""
    return [bits(pool.keys).clone(), bits(pool.values).clone(), pool.key_scales.cpu().clone(), pool.value_scales.cpu().clone()]


def check_pool(pool, want):
    for name, got, w in zip(("keys", "values", "key_scales", "value_scales"), parts(pool), want):
        assert torch.equal(got, w), (name, int((got != w).sum()), torch.nonzero(got != w)[:5].tolist())


def random_pool(dev, pages, kv_heads, page, d, dtype, seed, std=1.0):
    """A pool of what blocks of random rows are quantised to, of different sizes."""
    g = torch.Generator(dev).manual_seed(seed)
    pool = Fp8Pool.new(pages, kv_heads, page, d, dtype, dev)
    blocks = page // 16
    e = torch.randint(-3, 3, (2, pages, kv_heads, blocks), generator=g, device=dev) - 7
    pool.key_scales.copy_(e[0] + 127)
    pool.value_scales.copy_(e[1] + 127)
    for t in (pool.keys, pool.values):
        x = torch.randn(t.shape, generator=g, device=dev) * (100.0 * std)
        t.copy_(x.clamp(-448, 448).to(torch.float8_e4m3fn))
    return pool


def rotated(x, cos, sin, d):
    """In fp32 as the kernel does it: products rounded, then their sum."""
    x = x.float().cpu().view(x.shape[0], -1, d)
    c, s = (t.float().cpu().reshape(t.shape[0], 1, d) for t in (cos, sin))
    return x * c + x.roll(d // 2, -1) * s


def tables(rows, d, dtype, g, dev):
    ang = torch.rand(rows, 1, d // 2, generator=g) * 6
    return (torch.cat((ang.cos(), ang.cos()), -1).to(dtype).to(dev), torch.cat((-ang.sin(), ang.sin()), -1).to(dtype).to(dev))


def take(state, lens, heads, kv_heads, d, start, new, dev, extra=0):
    return page_tables(state, i32(start, dev), i32(new, dev), rows=sum(new) + extra, max_new=max(max(new), 1), heads=heads,
                       kv_heads=kv_heads, head_dim=d)


# ---------------------------------------------------------------- write
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,d,page,new,start,f32_tables,pad", [
    (4, 2, 64, 16, [1], [0], False, 0), (5, 1, 128, 16, [1, 0, 33, 2], [15, 9, 0, 31], False, 3),
    (8, 8, 64, 32, [70, 1, 7], [5, 200, 25], True, 0), (32, 8, 128, 16, [100, 1, 1, 13], [12, 40, 0, 3], True, 8),
    (2, 1, 128, 128, [300], [100], False, 1), (2, 1, 64, 1024, [500, 1, 300, 9], [3, 7, 1019, 15], False, 0),
    (1, 1, 128, 64, [1] * 190, list(range(190)), False, 0), (2, 2, 128, 16, [16, 17, 15, 1], [16, 15, 1, 31], False, 0),
    (2, 1, 64, 16, [600, 3], [0, 14], False, 5),
])
def test_write(dev, heads, kv_heads, d, page, new, start, f32_tables, pad, dtype):
    g = torch.Generator().manual_seed(sum(new) + d)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev)  # noqa: E731
    rows = sum(new) + 5  # five rows behind the last request's
    pages = sum(-(-(s + c) // page) for s, c in zip(start, new)) + 3
    state = PageState.new(len(new), max(s + c for s, c in zip(start, new)), pages, page, dev)
    state.free.copy_(i32(random.Random(d).sample(range(pages), pages), dev))
    step = take(state, None, heads, kv_heads, d, start, new, dev, extra=5)
    qkv = rn(rows, (heads + 2 * kv_heads) * d + pad)
    qkv[::3] *= 4  # rows that make exponents grow
    q, k, v = qkv[:, :heads * d], qkv[:, heads * d:(heads + kv_heads) * d], qkv[:, (heads + kv_heads) * d:(heads + 2 * kv_heads) * d]
    cos, sin = tables(rows, d, torch.float32 if f32_tables else dtype, g, dev)
    pool = random_pool(dev, pages, kv_heads, page, d, dtype, 1)
    want = parts(pool)
    fp8_ref.write(*want, rotated(k, cos, sin, d).double(), v.double().cpu().view(rows, kv_heads, d), step.slots.tolist(), dtype)
    before = q.clone()
    out = rotary_paged_write_fp8(q, k, v, cos, sin, pool, step)
    check_pool(pool, want)
    assert torch.equal(q, before)
    assert torch.equal(out.cpu(), rotated(q, cos, sin, d).to(dtype).view(rows, -1))
    # In place, and again: nothing more changes.
    assert rotary_paged_write_fp8(q, k, v, cos, sin, pool, step, out=q).data_ptr() == q.data_ptr()
    assert torch.equal(q, out)
    check_pool(pool, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 64])
def test_blocks_fill_while_requests_decode(dev, page, dtype):
    """Rows of very different sizes, one or a few a step, some taken back and written again: exponents grow, and earlier
    codes move with them."""
    rng, g = random.Random(page), torch.Generator().manual_seed(page)
    n, kv_heads, d = 6, 2, 64
    state = PageState.new(n, 200, 13 * n, page, dev)
    pool = random_pool(dev, 13 * n, kv_heads, page, d, dtype, 3)
    want, lens = parts(pool), [0] * n
    for _ in range(60):
        start = [max(0, s - rng.choice((0, 0, 0, 1, 3))) for s in lens]
        new = [rng.choice((0, 1, 1, 1, 4)) for _ in range(n)]
        rows = max(sum(new), 1)
        new[0] += rows - sum(new)
        step = take(state, None, 2, kv_heads, d, start, new, dev)
        size = torch.exp2(torch.randint(-12, 7, (rows, 1), generator=g).float())
        k, v = ((torch.randn(rows, kv_heads * d, generator=g) * size).to(dtype).to(dev) for _ in range(2))
        q = torch.randn(rows, 2 * d, generator=g).to(dtype).to(dev)
        cos, sin = tables(rows, d, dtype, g, dev)
        fp8_ref.write(*want, rotated(k, cos, sin, d).double(), v.double().cpu().view(rows, kv_heads, d), step.slots.tolist(), dtype)
        rotary_paged_write_fp8(q, k, v, cos, sin, pool, step)
        check_pool(pool, want)
        lens = [s + c for s, c in zip(start, new)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [16, 600])
def test_every_number_of_a_type_is_written(dev, rows, dtype):
    """All numbers of the type as values, blocks of one magnitude and of all, with NaN and infinities."""
    every = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    order = torch.argsort(torch.nan_to_num(every.float().abs(), nan=0.0))
    mixed = every[torch.randperm(65536, generator=torch.Generator().manual_seed(1))]
    d, state = 128, PageState.new(1, 1024, 64, 16, dev)
    for data in (every[order], mixed):
        for at in range(0, 65536, rows * d):
            v = data[at:at + rows * d].reshape(-1, d).to(dev)
            n = v.shape[0]
            page_tables(state, i32([0], dev), i32([0], dev), rows=0, max_new=0)
            step = take(state, None, 1, 1, d, [0], [n], dev)
            pool = random_pool(dev, 64, 1, 16, d, dtype, 2)
            want = parts(pool)
            one, zero = torch.ones(1, d, device=dev), torch.zeros(1, d, device=dev)
            # (k * 1 + rolled * 0 would be NaN beside an infinity: keys are the finite numbers)
            k = torch.where(torch.isfinite(v), v, 1.0)
            fp8_ref.write(*want, rotated(k, one, zero, d).double(), v.double().cpu().view(n, 1, d), step.slots.tolist(), dtype)
            rotary_paged_write_fp8(torch.zeros_like(v), k, v, one, zero, pool, step)
            got = parts(pool)
            for a in (0, 1):  # a NaN's sign is of no consequence
                both = ((got[a] & 127) == 127) & ((want[a] & 127) == 127)
                assert torch.equal(torch.where(both, 0, got[a]), torch.where(both, 0, want[a])), (at, int((got[a] != want[a]).sum()))
            assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
            kd, vd = pool.dequantize()
            assert bool(torch.isfinite(kd[:n // 16 + 1]).all()) and not bool(torch.isinf(vd).any())


def test_rows_without_a_slot(dev):
    """A pool that runs short: tokens without a page are rotated and not written."""
    state = PageState.new(2, 64, 3, 16, dev)
    step = take(state, None, 2, 1, 64, [0, 0], [30, 30], dev)
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(60, w, generator=g).half().to(dev) for w in (128, 64, 64))
    cos, sin = tables(60, 64, torch.float16, g, dev)
    pool = random_pool(dev, 3, 1, 16, 64, torch.float16, 1)
    want = parts(pool)
    slots = step.slots.tolist()
    assert slots[46:] == [-1] * 14
    fp8_ref.write(*want, rotated(k, cos, sin, 64).double(), v.double().cpu().view(60, 1, 64), slots, torch.float16)
    out = rotary_paged_write_fp8(q, k, v, cos, sin, pool, step)
    check_pool(pool, want)
    assert torch.equal(out.cpu(), rotated(q, cos, sin, 64).half().view(60, -1))


# ---------------------------------------------------------------- attention
def cache_case(dev, new, start, heads, kv_heads, d, page, dtype, seed, spare=3, extra_rows=0, std=1.5):
    g = torch.Generator(dev).manual_seed(seed)
    need = [-(-(s + c) // page) for s, c in zip(start, new)]
    pages = sum(need) + spare
    table, free = ref.draw_table(need, pages, seed)
    state = PageState(table=table.to(dev), held=i32(need, dev), free=i32(free + [-1] * (pages - len(free)), dev),
                      counts=i32([len(free), 0], dev), page=page)
    step = take(state, None, heads, kv_heads, d, start, new, dev, extra=extra_rows)
    q = torch.randn(sum(new) + extra_rows, heads * d, generator=g, device=dev).to(dtype) * std
    return q, random_pool(dev, pages, kv_heads, page, d, dtype, seed), table, step


def check_attention(got, q, pool, table, start, new, scale):
    rows = sum(new)
    keys, values = pool.dequantize()
    want, spread = ref.attention(q[:rows], keys, values, table, start, new, scale)
    longest = max(s + c for s, c in zip(start, new))
    err = (got[:rows].double() - want).abs()
    ok = err <= ref.bound(want, spread, pool.dtype, longest, scale_of_scores=160.0)
    assert bool(ok.all()), (float(err.max()), int((~ok).sum()))


CASES = [
    # new, start, heads, kv_heads, d, page
    ([1], [0], 1, 1, 64, 16), ([1], [14], 4, 2, 64, 16), ([1], [15], 4, 2, 64, 16), ([1], [16], 4, 1, 128, 16),
    ([1, 0, 1, 1], [31, 5, 32, 33], 8, 2, 128, 16), ([1] * 5, [63, 64, 65, 127, 128], 32, 8, 128, 32),
    ([1, 1], [255, 256], 5, 1, 128, 16), ([1, 1, 1], [257, 511, 700], 28, 4, 128, 128), ([1], [3000], 8, 1, 128, 16),
    ([5, 3, 9], [100, 0, 37], 16, 4, 128, 16), ([2, 17, 1], [1, 300, 0], 12, 2, 64, 16), ([4], [0], 32, 1, 64, 16),
    ([33], [0], 4, 4, 64, 16), ([64, 1, 130], [0, 800, 65], 8, 2, 128, 64), ([300, 1, 1], [0, 40, 513], 8, 1, 64, 16),
    ([129, 127, 128], [0, 1, 500], 8, 8, 128, 16), ([200], [1500], 16, 2, 128, 1024), ([31] * 3, [1, 2, 3], 3, 1, 64, 32),
    ([7, 1], [2000, 9000], 8, 2, 128, 16), ([1] * 130, [3 * i for i in range(130)], 4, 2, 64, 16),
    ([513, 90], [0, 4000], 32, 8, 128, 16), ([48, 1, 48], [0, 0, 2], 40, 1, 64, 16), ([1, 1, 2], [191, 192, 383], 16, 2, 64, 64),
    ([8, 8], [300, 1000], 4, 1, 128, 16), ([8, 5], [47, 1000], 4, 1, 64, 32),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new,start,heads,kv_heads,d,page", CASES)
def test_attention(dev, new, start, heads, kv_heads, d, page, dtype):
    q, pool, table, step = cache_case(dev, new, start, heads, kv_heads, d, page, dtype, sum(start) + heads)
    got = paged_attention_fp8(q, pool, step, d ** -0.5)
    check_attention(got, q, pool, table, start, new, d ** -0.5)
    assert torch.equal(paged_attention_fp8(q, pool, step, d ** -0.5), got)


@pytest.mark.parametrize("seed", range(12))
def test_attention_random_shapes(dev, seed):
    rng = random.Random(seed)
    heads, kv_heads, d = rng.choice(((32, 8, 128), (16, 4, 128), (4, 2, 64), (8, 8, 64), (12, 2, 64), (28, 4, 128), (32, 2, 64)))
    n = rng.choice((1, 2, 7, 40))
    new = [rng.choice((0, 1, 1, rng.randint(2, 9), rng.randint(10, 400 // n + 10))) for _ in range(n)]
    new[0] = max(new[0], 1)
    start = [rng.choice((0, rng.randint(0, 60), rng.randint(0, 2500))) for _ in range(n)]
    q, pool, table, step = cache_case(dev, new, start, heads, kv_heads, d, rng.choice((16, 32, 64, 256)), rng.choice(DTYPES), seed)
    check_attention(paged_attention_fp8(q, pool, step, d ** -0.5), q, pool, table, start, new, d ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 200])
def test_every_code_and_exponent_is_read_exactly(dev, rows, dtype):
    """A first token attends to itself alone: its result is its values."""
    d, page = 128, 16
    lo, hi = fp8_ref.RANGE[dtype]
    state = PageState.new(1, 256, 16, page, dev)
    step = take(state, None, 1, 1, d, [0], [rows], dev)
    pg = int(state.table[0, 0])
    q = torch.randn(rows, d, device=dev).to(dtype)
    pool = Fp8Pool.new(16, 1, page, d, dtype, dev)
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[(codes & 127) != 127]
    for e in range(lo, hi + 1):
        usable = codes if e < hi else codes[(codes & 127) <= int(fp8_ref.encode(torch.tensor(240.0).double()))]
        for at in range(0, len(usable), d):
            c = usable[at:at + d]
            c = torch.cat((c, torch.zeros(d - len(c), dtype=torch.uint8)))
            pool.values.view(torch.uint8)[pg, 0, :, 0] = c.to(dev)
            pool.value_scales[pg, 0, 0] = e + 127
            want = fp8_ref.decode(c) * 2.0 ** e
            assert torch.equal(want, want.to(dtype).double())  # a number of the type
            got = paged_attention_fp8(q, pool, step, 0.1)[0].cpu().double()
            assert torch.equal(got, want), e


@pytest.mark.parametrize("new,start", [([1, 1], [40, 300]), ([20, 3], [7, 600]), ([150, 1], [33, 30]),
                                       ([3, 1], [1300, 90])])
@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_behind_a_row_reaches_it(dev, new, start, dtype):
    """NaN codes and exponents of infinity in the free pages, behind the requests' ends and in later tokens of a chunk."""
    heads, kv_heads, d, page = 8, 2, 128, 32
    q, pool, table, step = cache_case(dev, new, start, heads, kv_heads, d, page, dtype, 5)
    want = paged_attention_fp8(q, pool, step, d ** -0.5)
    used = torch.zeros(pool.shape[0], page, dtype=torch.bool, device=dev)
    for i, (s, c) in enumerate(zip(start, new)):
        at = torch.arange(s + c, device=dev)
        used[table[i].to(dev).long()[at // page], at % page] = True
    hidden = (~used)[:, None].expand(-1, kv_heads, -1)
    pool.keys.view(torch.uint8)[hidden] = 0x7f
    pool.values.view(torch.uint8).transpose(2, 3)[hidden] = 0xff
    blocks = ~used.view(-1, page // 16, 16).any(-1)[:, None].expand(-1, kv_heads, -1)
    for byte in (0, 255):
        pool.key_scales[blocks] = byte
        pool.value_scales[blocks] = byte
        assert torch.equal(paged_attention_fp8(q, pool, step, d ** -0.5), want)
    if new[0] > 2:
        # The last token of the first request: only its own row sees it.
        p = start[0] + new[0] - 1
        pg, off = int(table[0, p // page]), p % page
        pool.keys.view(torch.uint8)[pg, :, off, 3] = 0x7f
        pool.values.view(torch.uint8)[pg, 0, 5, off] = 0xff
        got = paged_attention_fp8(q, pool, step, d ** -0.5)
        r = new[0] - 1
        assert torch.equal(got[:r], want[:r]) and torch.equal(got[r + 1:], want[r + 1:])
        assert bool(got[r].isnan().all())


@pytest.mark.parametrize("rows", [1, 40])
def test_nan_values_reach_the_rows_that_see_them(dev, rows):
    start, d = 50, 64
    q, pool, table, step = cache_case(dev, [rows], [start], 4, 2, d, 16, torch.float16, 9)
    at = [p for p in (3, 17, 60, 89) if p < start + rows]
    for p in at:
        pool.values.view(torch.uint8)[int(table[0, p // 16]), 0, p % 64, p % 16] = 0x7f
    got = paged_attention_fp8(q, pool, step, d ** -0.5).view(rows, 4, d)
    for p in at:
        sees = torch.arange(rows, device=dev) + start >= p
        assert bool(got[sees][:, :2, p % 64].isnan().all())
        assert bool(got[~sees][:, :, p % 64].isfinite().all())
    assert bool(got[:, 2:].isfinite().all())


@pytest.mark.parametrize("new,start", [([1], [70]), ([50], [70]), ([1], [1500])])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales_that_are_not_positive(dev, new, start, scale):
    q, pool, table, step = cache_case(dev, new, start, 4, 2, 64, 16, torch.bfloat16, 2)
    check_attention(paged_attention_fp8(q, pool, step, scale), q, pool, table, start, new, scale)


def test_rows_behind_the_last_request_are_left(dev):
    q, pool, table, step = cache_case(dev, [3, 1], [0, 20], 4, 2, 64, 16, torch.float16, 3, extra_rows=30)
    out = torch.full_like(q, 7.0)
    assert paged_attention_fp8(q, pool, step, 0.125, out=out) is out
    assert bool((out[4:] == 7.0).all())
    check_attention(out, q, pool, table, [0, 20], [3, 1], 0.125)


def test_strided_rows_pages_and_outputs(dev):
    d, new, start, dt = 64, [9, 1], [30, 70], torch.bfloat16
    q, pool, table, step = cache_case(dev, new, start, 4, 2, d, 16, dt, 4)
    want = paged_attention_fp8(q, pool, step, 0.125)
    wide = torch.zeros(q.shape[0], q.shape[1] + 24, device=dev, dtype=dt)
    wide[:, 8:8 + q.shape[1]] = q
    pages = pool.shape[0]
    layers = torch.zeros(pages, 3, *pool.shape[1:], dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)  # three layers, page by page
    vlayers = layers.clone().view(pages, 3, 2, d, 16)
    layers[:, 1].view(torch.uint8).copy_(pool.keys.view(torch.uint8))
    vlayers[:, 1].view(torch.uint8).copy_(pool.values.view(torch.uint8))
    apart = Fp8Pool(layers[:, 1], vlayers[:, 1], pool.key_scales, pool.value_scales, dt)
    out = torch.zeros_like(wide)
    paged_attention_fp8(wide[:, 8:8 + q.shape[1]], apart, step, 0.125, out=out[:, 16:16 + q.shape[1]])
    assert torch.equal(out[:, 16:16 + q.shape[1]], want)
    assert not out[:, :16].any() and not out[:, 16 + q.shape[1]:].any()
    wide[:, 1:1 + q.shape[1]] = q
    assert torch.equal(paged_attention_fp8(wide[:, 1:1 + q.shape[1]], apart, step, 0.125), want)  # not 16-byte aligned
    k = torch.randn(10, 2 * d, device=dev).to(dt)
    one, zero = torch.ones(1, d, device=dev, dtype=dt), torch.zeros(1, d, device=dev, dtype=dt)
    expect = parts(pool)
    fp8_ref.write(*expect, k.double().cpu().view(10, 2, d), k.double().cpu().view(10, 2, d), step.slots.tolist(), dt)
    rotary_paged_write_fp8(q, k, k, one, zero, apart, step)
    assert torch.equal(bits(layers)[:, 1], expect[0]) and torch.equal(bits(vlayers)[:, 1], expect[1])
    assert not bits(layers)[:, ::2].any() and not bits(vlayers)[:, ::2].any()


def test_pages_outside_the_pool_give_nan_to_the_rows_that_need_them(dev):
    for new, start in (([6, 1], [30, 40]), ([60, 1], [30, 40])):
        q, pool, table, step = cache_case(dev, new, start, 4, 2, 64, 16, torch.bfloat16, 6)
        want = paged_attention_fp8(q, pool, step, 0.125)
        for bad in (-1, pool.shape[0], 2 ** 31 - 1, -2 ** 31):
            step.state.table[0, 2] = bad     # positions 32 to 47: rows 2 and on of the first request
            got = paged_attention_fp8(q, pool, step, 0.125)
            n = new[0]
            assert torch.equal(got[:2], want[:2]) and bool(got[2:n].isnan().all()) and torch.equal(got[n:], want[n:])


def test_large_pool_offsets_pass_32_bits(dev):
    """A pool of more than 2^32 bytes: the last pages are read and written where they are."""
    d, page, kv = 128, 16, 8
    pages = 2 ** 32 // (kv * page * d) + 40
    pool = Fp8Pool.new(pages, kv, page, d, torch.bfloat16, dev)
    ids = [pages - 1, 0, pages - 2, 5]
    state = PageState(table=i32([ids], dev), held=i32([4], dev), free=i32([0] * pages, dev), counts=i32([0, 0], dev), page=page)
    g = torch.Generator(dev).manual_seed(1)
    q, k, v = (torch.randn(50, 1024, generator=g, device=dev).bfloat16() for _ in range(3))
    cos, sin = torch.ones(1, d, device=dev).bfloat16(), torch.zeros(1, d, device=dev).bfloat16()
    step = take(state, None, 8, 8, d, [0], [50], dev)
    rotary_paged_write_fp8(q, k, v, cos, sin, pool, step)
    few = [t[ids] for t in (pool.keys.view(torch.uint8), pool.values.view(torch.uint8), pool.key_scales, pool.value_scales)]
    small = Fp8Pool(few[0].view(torch.float8_e4m3fn), few[1].view(torch.float8_e4m3fn), few[2], few[3], torch.bfloat16)
    want = parts(Fp8Pool.new(4, kv, page, d, torch.bfloat16, dev))
    fp8_ref.write(*want, k.double().cpu().view(50, 8, d), v.double().cpu().view(50, 8, d), list(range(50)), torch.bfloat16)
    check_pool(small, want)
    got = paged_attention_fp8(q, pool, step, d ** -0.5)
    check_attention(got, q, small, torch.tensor([[0, 1, 2, 3]]), [0], [50], d ** -0.5)
    one = take(state, None, 8, 8, d, [49], [1], dev)
    got = paged_attention_fp8(q[49:], pool, one, d ** -0.5)
    check_attention(got, q[49:], small, torch.tensor([[0, 1, 2, 3]]), [49], [1], d ** -0.5)


# ---------------------------------------------------------------- graphs, streams, refusals
@pytest.mark.parametrize("longest", [300, 2000])
def test_steps_captured_and_replayed(dev, longest):
    """Tables, write and attention of one step in a graph, replayed as the requests grow."""
    n, heads, kv_heads, d, page, dt = 5, 8, 2, 64, 16, torch.bfloat16
    width = -(-longest // page)
    state = PageState.new(n, longest, n * width, page, dev)
    pool = random_pool(dev, n * width, kv_heads, page, d, dt, 1)
    step = PagedStep(state, n, 1, heads, kv_heads, d)
    lens, one = i32([3, longest - 40, 17, 0, 100], dev), i32([1] * n, dev)
    qkv = torch.randn(n, (heads + 2 * kv_heads) * d, device=dev).to(dt)
    q, k, v = qkv.split((heads * d, kv_heads * d, kv_heads * d), dim=1)
    cos, sin = torch.rand(1, d, device=dev).to(dt), torch.rand(1, d, device=dev).to(dt)

    def run():
        page_tables(state, lens, one, step=step)
        r = rotary_paged_write_fp8(q, k, v, cos, sin, pool, step)
        return paged_attention_fp8(r, pool, step, 0.125)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run()
    for turn in range(20):
        qkv.copy_(torch.randn(qkv.shape, device=dev) * (1 + turn % 3))
        mine = parts(pool)
        graph.replay()
        torch.cuda.synchronize()
        fp8_ref.write(*mine, rotated(k, cos, sin, d).double(), v.double().cpu().view(n, kv_heads, d), step.slots.tolist(), dt)
        check_pool(pool, mine)
        rot = rotated(q, cos, sin, d).to(dt).view(n, -1).to(dev)
        check_attention(out, rot, pool, state.table.cpu(), lens.tolist(), [1] * n, 0.125)
        lens.add_(1)


def test_two_steps_of_one_state_on_two_streams(dev):
    q, pool, table, a = cache_case(dev, [1, 1, 1], [3000, 40, 900], 8, 2, 128, 16, torch.bfloat16, 11)
    b = take(a.state, None, 8, 2, 128, [3000, 40, 900], [1, 1, 1], dev)
    want = paged_attention_fp8(q, pool, a, 0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(10):
        for s, step in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                outs.append(paged_attention_fp8(q, pool, step, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_a_step_that_was_only_recorded(dev):
    """Whatever the memory of a step's tables holds, the calls keep to their tensors."""
    new, start = [1, 1, 1], [900, 300, 77]
    q, pool, table, eager = cache_case(dev, new, start, 8, 2, 128, 16, torch.bfloat16, 1)
    step = PagedStep(eager.state, 3, 1, 8, 2, 128)
    graph = torch.cuda.CUDAGraph()
    first, more = i32(start, dev), i32(new, dev)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        page_tables(eager.state, first, more, step=step)
    out = torch.full_like(q, 7.0)
    k = torch.randn(3, 256, device=dev).bfloat16()
    cos = torch.ones(1, 128, device=dev).bfloat16()
    before = parts(pool)
    for junk in (-1, 2 ** 31 - 1, -2 ** 31, 1 << 24):
        step._ints.fill_(junk)
        paged_attention_fp8(q, pool, step, 0.1, out=out)
        assert bool((out == 7.0).all())
        rotary_paged_write_fp8(q, k, k, cos, cos, pool, step)
        check_pool(pool, before)


@pytest.mark.parametrize("native", [True, False])
def test_what_torch_has_to_see_is_refused(dev, monkeypatch, native):
    q, pool, table, step = cache_case(dev, [3, 1], [0, 20], 4, 2, 64, 16, torch.float16, 3)
    k, cos = torch.randn(4, 128, device=dev).half(), torch.randn(4, 64, device=dev).half()
    if not native:
        none = lambda *a: None  # noqa: E731
        monkeypatch.setattr(_ffi, "calls", lambda: SimpleNamespace(page_tables=none, paged_write8=none, paged_attention8=none))

    def attend(q, out=None):
        return paged_attention_fp8(q, pool, step, 0.125, out=out)

    def write(q, k=k, v=k, cos=cos, out=None):
        return rotary_paged_write_fp8(q, k, v, cos, cos, pool, step, out=out)

    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: attend(dual(q)), lambda: write(dual(q)), lambda: write(q, k=dual(k)), lambda: write(q, v=dual(k)),
                     lambda: write(q, cos=dual(cos))):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
    for f in (attend, write):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(lambda x: f(x), (q,), check_trace=False)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda x: f(x))(q)
        with pytest.raises(RuntimeError, match="no backward pass"):
            f(q.clone().requires_grad_())
        with pytest.raises(RuntimeError, match="no backward pass"):
            f(q, out=torch.ones_like(q, requires_grad=True))
        out, w = torch.ones_like(q), torch.ones_like(q, requires_grad=True)
        y = w * out
        assert f(q, out=out) is out
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        with torch.inference_mode():
            inside = torch.ones_like(q)
            f(q, out=inside)
        with pytest.raises(RuntimeError, match="inference mode"):
            f(q, out=inside)


@pytest.mark.parametrize("native", [True, False])
def test_calls_that_do_not_fit_are_refused(dev, monkeypatch, native):
    q, pool, table, step = cache_case(dev, [3, 1], [0, 20], 4, 2, 64, 16, torch.float16, 3)
    if not native:
        none = lambda *a: None  # noqa: E731
        monkeypatch.setattr(_ffi, "calls", lambda: SimpleNamespace(page_tables=none, paged_write8=none, paged_attention8=none))
    k, cos = torch.randn(4, 128, device=dev).half(), torch.randn(4, 64, device=dev).half()
    pages = pool.shape[0]
    other = Fp8Pool.new(pages, 2, 32, 64, torch.float16, dev)   # pages of another size
    few = Fp8Pool.new(pages - 1, 2, 16, 64, torch.float16, dev)
    for bad in (other, few):
        with pytest.raises(ValueError):
            paged_attention_fp8(q, bad, step, 0.1)
        with pytest.raises(ValueError):
            rotary_paged_write_fp8(q, k, k, cos, cos, bad, step)
    for x in (q.bfloat16(), q[:3], q[:, :64], q.float()):
        with pytest.raises(ValueError):
            paged_attention_fp8(x, pool, step, 0.1)
    with pytest.raises(ValueError):
        rotary_paged_write_fp8(q.bfloat16(), k, k, cos, cos, pool, step)
    with pytest.raises(ValueError):
        rotary_paged_write_fp8(q, k[:, :64], k, cos, cos, pool, step)
    with pytest.raises(ValueError):
        rotary_paged_write_fp8(q[:3], k[:3], k[:3], cos[:3], cos[:3], pool, step)
    empty = PagedStep(step.state, 4, 3, 4, 2, 64)
    with pytest.raises(ValueError, match="page_tables fills it"):
        paged_attention_fp8(q, pool, empty, 0.1)
    with pytest.raises(ValueError, match="page_tables fills it"):
        rotary_paged_write_fp8(q, k, k, cos, cos, pool, empty)
    bare = page_tables(step.state, i32([0, 20], dev), i32([3, 1], dev), rows=4, max_new=3)
    with pytest.raises(ValueError, match="work list"):
        paged_attention_fp8(q, pool, bare, 0.1)
    rotary_paged_write_fp8(q, k, k, cos, cos, pool, bare)  # the write needs none
