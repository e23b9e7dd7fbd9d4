"""The paged KV cache's operators (GPU) against plain 64-bit forms, at the sizes and masks where they can go wrong."""

import random
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from multi_lora_amd import _ffi
from multi_lora_amd.kernels import PagedStep, PageState, page_tables, paged_attention, rotary_paged_write, verify_drafts

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# ---------------------------------------------------------------- page tables
def check_step(state, sim, step, want, rows):
    indptr, lens, pos, slots, missing = want
    assert step.row_indptr.tolist() == indptr and step.kv_lens.tolist() == lens
    assert step.positions.tolist() == pos and step.slots.tolist() == slots
    assert state.held.tolist() == sim.held
    assert state.counts.tolist() == [len(sim.stack), missing]
    assert state.free[:len(sim.stack)].tolist() == sim.stack
    table = state.table.tolist()
    for i, k in enumerate(sim.held):
        assert table[i][:k] == sim.table[i][:k]


@pytest.mark.parametrize("n,page,longest,pool,seed", [
    (1, 8, 60, 9, 0), (3, 16, 200, 40, 1), (70, 16, 90, 500, 2), (1030, 32, 70, 2600, 3), (2100, 8, 20, 3000, 4),
    (64, 1024, 5000, 300, 5),
])
def test_page_tables_over_steps(dev, n, page, longest, pool, seed):
    """Requests come, grow, take tokens back and go; some calls find the pool short."""
    rng = random.Random(seed)
    width = -(-longest // page)
    state, sim = PageState.new(n, longest, pool, page, dev), ref.Pages(n, width, pool, page)
    lens = [0] * n
    for _ in range(6):
        start, new = [], []
        for i in range(n):
            kind = rng.random()
            s = 0 if kind < 0.2 else max(0, lens[i] - rng.randint(0, 5)) if kind < 0.5 else lens[i]
            c = 0 if kind < 0.1 else 1 if kind < 0.7 else rng.randint(0, longest - s)
            start.append(s)
            new.append(min(c, longest - s))
        rows = sum(new) + rng.choice((0, 1, 300))
        step = page_tables(state, i32(start, dev), i32(new, dev), rows=rows, max_new=max(new))
        check_step(state, sim, step, sim.step(start, new, rows), rows)
        lens = [s + c for s, c in zip(start, new)]


def test_page_tables_give_back_restores_the_stack(dev):
    state = PageState.new(5, 400, 60, 16, dev)
    state.free.copy_(i32(random.Random(1).sample(range(60), 60), dev))
    page_tables(state, i32([0] * 5, dev), i32([30, 0, 17, 1, 64], dev), rows=112, max_new=64)
    before = state.free[:int(state.counts[0])].tolist()
    page_tables(state, i32([30, 0, 17, 1, 64], dev), i32([100, 5, 0, 31, 0], dev), rows=136, max_new=100)
    page_tables(state, i32([30, 0, 17, 1, 64], dev), i32([0] * 5, dev), rows=0, max_new=0)
    assert state.free[:int(state.counts[0])].tolist() == before


def test_page_tables_past_the_table_and_bad_lengths(dev):
    """Positions past the table's width have no slot; negative lengths count as none."""
    state = PageState.new(3, 32, 8, 16, dev)
    step = page_tables(state, i32([0, -7, 30], dev), i32([40, 2, -1], dev), rows=64, max_new=40)
    assert step.row_indptr.tolist() == [0, 40, 42, 42] and step.kv_lens.tolist() == [40, 2, 30]
    slots = step.slots.tolist()
    assert all(s >= 0 for s in slots[:32]) and slots[32:40] == [-1] * 8 and all(s >= 0 for s in slots[40:42])
    assert slots[42:] == [-1] * 22 and step.positions.tolist()[40:] == [0, 1] + [0] * 22
    assert state.held.tolist() == [2, 1, 2]


@pytest.mark.parametrize("n", [3, 1200])  # one launch, and two
def test_bounds_that_are_too_small_are_kept(dev, n):
    """Rows and new tokens past the step's bounds are not given out, and what is given fits together."""
    state = PageState.new(n, 64, 16 + n, 16, dev)
    zeros = [0] * (n - 3)
    step = page_tables(state, i32([7, 20, 0] + zeros, dev), i32([10, 12, 10] + zeros, dev), rows=15, max_new=11,
                       heads=2, kv_heads=1, head_dim=64)
    assert step.row_indptr.tolist() == [0, 10] + [15] * (n - 1) and step.kv_lens.tolist() == [17, 25, 0] + zeros
    assert step.positions.tolist() == list(range(7, 17)) + list(range(20, 25))
    step = page_tables(state, i32([7, 20, 0] + zeros, dev), i32([10, 12, 10] + zeros, dev), rows=40, max_new=11)
    assert step.row_indptr.tolist()[:4] == [0, 10, 21, 31] and step.kv_lens.tolist()[:3] == [17, 31, 10]


@pytest.mark.parametrize("n", [5, 1100])
def test_a_step_continues_from_its_own_lengths(dev, n):
    """start_lens is the step's kv_lens, which the call rewrites."""
    state, sim = PageState.new(n, 400, 26 * n, 16, dev), ref.Pages(n, 25, 26 * n, 16)
    new = [1 + i % 3 for i in range(n)]
    step = page_tables(state, i32([0] * n, dev), i32(new, dev), rows=sum(new), max_new=3)
    check_step(state, sim, step, sim.step([0] * n, new, sum(new)), sum(new))
    for turn in range(1, 20):
        page_tables(state, step.kv_lens, i32(new, dev), step=step)
        check_step(state, sim, step, sim.step([turn * c for c in new], new, sum(new)), sum(new))


# ---------------------------------------------------------------- rotary and write
def half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,d,page,new,start,f32_tables,pad", [
    (4, 2, 64, 8, [1], [0], False, 0), (5, 1, 128, 16, [1, 0, 33, 2], [15, 9, 0, 31], False, 3),
    (8, 8, 64, 32, [70, 1, 7], [5, 200, 25], True, 0), (32, 8, 128, 16, [100, 1, 1, 13], [12, 40, 0, 3], True, 8),
    (2, 1, 128, 128, [300], [100], False, 1),
    (2, 1, 64, 8, [1500, 1, 700, 9], [3, 7, 8, 15], False, 0), (1, 1, 128, 64, [1] * 190, list(range(190)), False, 0),
])
def test_rotary_paged_write(dev, heads, kv_heads, d, page, new, start, f32_tables, pad, dtype):
    g = torch.Generator().manual_seed(sum(new) + d)
    rn = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev)  # noqa: E731
    rows = sum(new) + 5  # five rows behind the last request's
    pages = sum(-(-(s + c) // page) for s, c in zip(start, new)) + 3
    state = PageState.new(len(new), max(s + c for s, c in zip(start, new)), pages, page, dev)
    state.free.copy_(i32(random.Random(d).sample(range(pages), pages), dev))
    step = page_tables(state, i32(start, dev), i32(new, dev), rows=rows, max_new=max(new))
    qkv = rn(rows, (heads + 2 * kv_heads) * d + pad)
    q, k, v = qkv[:, :heads * d], qkv[:, heads * d:(heads + kv_heads) * d], qkv[:, (heads + kv_heads) * d:(heads + 2 * kv_heads) * d]
    ang = torch.rand(rows, 1, d // 2, generator=g) * 6
    tab = torch.float32 if f32_tables else dtype
    cos = torch.cat((ang.cos(), ang.cos()), -1).to(tab).to(dev)
    sin = torch.cat((-ang.sin(), ang.sin()), -1).to(tab).to(dev)
    keys, values = rn(pages, kv_heads, page, d), rn(pages, kv_heads, d, page)
    want_k, want_v = keys.double(), values.double()
    rot = lambda t: t.double().view(rows, -1, d) * cos.double() + t.double().view(rows, -1, d).roll(d // 2, -1) * sin.double()  # noqa: E731
    at = step.slots.tolist()
    touched = torch.zeros(pages, kv_heads, page, dtype=torch.bool)
    for r, slot in enumerate(at):
        if slot >= 0:
            want_k[slot // page, :, slot % page] = rot(k)[r]
            want_v[slot // page, :, :, slot % page] = v[r].double().view(kv_heads, d)
            touched[slot // page, :, slot % page] = True
    old = keys.clone()
    out = rotary_paged_write(q, k, v, cos, sin, keys, values, step.slots)
    # One rounding of x cos + y sin; its fp32 terms (two products and a sum) are off by 3 * 2^-24 of |x cos| + |y sin| <= 12.
    tol = lambda w: half_step(dtype) * w.abs() + 36 * 2.0 ** -24  # noqa: E731
    qw = rot(q).reshape(rows, -1)
    assert bool(((out.double() - qw).abs() <= tol(qw)).all())
    assert bool(((keys.double() - want_k).abs() <= tol(want_k)).all())
    assert torch.equal(keys.cpu()[~touched], old.cpu()[~touched])
    assert torch.equal(values.double(), want_v)
    again = q.clone()
    assert rotary_paged_write(again, k, v, cos, sin, keys, values, step.slots, out=again) is again
    assert torch.equal(again, out)


def test_rotary_paged_write_one_table_row_and_slots_outside(dev):
    q = torch.randn(3, 128, device=dev).half()
    kv = torch.randn(3, 64, device=dev).half()
    cos, sin = torch.ones(1, 64, device=dev).half(), torch.zeros(1, 64, device=dev).half()
    keys, values = torch.zeros(2, 1, 8, 64, device=dev).half(), torch.zeros(2, 1, 64, 8, device=dev).half()
    out = rotary_paged_write(q, kv, kv, cos, sin, keys, values, i32([16, -1, 9], dev))
    assert torch.equal(out, q)
    assert torch.equal(keys[1, 0, 1], kv[2]) and torch.equal(values[1, 0, :, 1], kv[2])
    assert int((keys != 0).any(-1).sum()) == 1


# ---------------------------------------------------------------- attention
def cache_case(dev, new, start, heads, kv_heads, d, page, dtype, seed, spare=3, extra_rows=0, std=1.5):
    g = torch.Generator(dev).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev).to(dtype)  # noqa: E731
    need = [-(-(s + c) // page) for s, c in zip(start, new)]
    pages = sum(need) + spare
    table, free = ref.draw_table(need, pages, seed)
    state = PageState(table=table.to(dev), held=i32(need, dev), free=i32(free + [-1] * (pages - len(free)), dev),
                      counts=i32([len(free), 0], dev), page=page)
    rows = sum(new) + extra_rows
    step = page_tables(state, i32(start, dev), i32(new, dev), rows=rows, max_new=max(new), heads=heads,
                       kv_heads=kv_heads, head_dim=d)
    q = rn(rows, heads * d) * std
    return q, rn(pages, kv_heads, page, d), rn(pages, kv_heads, d, page), table, step


def check_attention(got, q, keys, values, table, start, new, scale, dtype):
    rows = sum(new)
    want, spread = ref.attention(q[:rows], keys, values, table, start, new, scale)
    longest = max(s + c for s, c in zip(start, new))
    err = (got[:rows].double() - want).abs()
    ok = err <= ref.bound(want, spread, dtype, longest)
    assert bool(ok.all()), (float(err.max()), int((~ok).sum()))


CASES = [
    # new, start, heads, kv_heads, d, page
    ([1], [0], 1, 1, 64, 8), ([1], [6], 4, 2, 64, 8), ([1], [7], 4, 2, 64, 8), ([1], [8], 4, 1, 128, 16),
    ([1, 0, 1, 1], [31, 5, 32, 33], 8, 2, 128, 16), ([1] * 5, [63, 64, 65, 127, 128], 32, 8, 128, 32),
    ([1, 1], [255, 256], 5, 1, 128, 16), ([1, 1, 1], [257, 511, 700], 28, 4, 128, 128), ([1], [3000], 8, 1, 128, 16),
    ([5, 3, 9], [100, 0, 37], 16, 4, 128, 16), ([2, 17, 1], [1, 300, 0], 12, 2, 64, 8), ([4], [0], 32, 1, 64, 16),
    ([33], [0], 4, 4, 64, 8), ([64, 1, 130], [0, 800, 65], 8, 2, 128, 64), ([300, 1, 1], [0, 40, 513], 8, 1, 64, 16),
    ([129, 127, 128], [0, 1, 500], 8, 8, 128, 16), ([200], [1500], 16, 2, 128, 1024), ([31] * 3, [1, 2, 3], 3, 1, 64, 32),
    ([7, 1], [2000, 9000], 8, 2, 128, 16), ([1] * 130, [3 * i for i in range(130)], 4, 2, 64, 16),
    ([513, 90], [0, 4000], 32, 8, 128, 16), ([48, 1, 48], [0, 0, 2], 40, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,start,heads,kv_heads,d,page", CASES)
def test_paged_attention(dev, new, start, heads, kv_heads, d, page, dtype):
    q, keys, values, table, step = cache_case(dev, new, start, heads, kv_heads, d, page, dtype, sum(start) + heads)
    got = paged_attention(q, keys, values, step, d ** -0.5)
    check_attention(got, q, keys, values, table, start, new, d ** -0.5, dtype)
    assert torch.equal(paged_attention(q, keys, values, step, d ** -0.5), got)


@pytest.mark.parametrize("seed", range(12))
def test_paged_attention_random_shapes(dev, seed):
    rng = random.Random(seed)
    heads, kv_heads, d = rng.choice(((32, 8, 128), (16, 4, 128), (4, 2, 64), (8, 8, 64), (12, 2, 64), (28, 4, 128), (32, 2, 64)))
    n = rng.choice((1, 2, 7, 40))
    new = [rng.choice((0, 1, 1, rng.randint(2, 9), rng.randint(10, 400 // n + 10))) for _ in range(n)]
    new[0] = max(new[0], 1)
    start = [rng.choice((0, rng.randint(0, 60), rng.randint(0, 2500))) for _ in range(n)]
    dtype = rng.choice((torch.bfloat16, torch.float16))
    page = rng.choice((8, 16, 64, 256))
    q, keys, values, table, step = cache_case(dev, new, start, heads, kv_heads, d, page, dtype, seed)
    got = paged_attention(q, keys, values, step, d ** -0.5)
    check_attention(got, q, keys, values, table, start, new, d ** -0.5, dtype)


@pytest.mark.parametrize("new,start", [([1, 1], [40, 300]), ([20, 3], [7, 600]), ([150, 1], [33, 30]),
                                       ([3, 1], [1300, 90])])
def test_nothing_behind_a_row_reaches_it(dev, new, start):
    """NaN and infinities in the free pages, in the pages behind the requests' ends and in later tokens of a chunk."""
    dtype, heads, kv_heads, d, page = torch.bfloat16, 8, 2, 128, 32
    q, keys, values, table, step = cache_case(dev, new, start, heads, kv_heads, d, page, dtype, 5)
    want = paged_attention(q, keys, values, step, d ** -0.5)
    used = torch.zeros(keys.shape[0], page, dtype=torch.bool, device=dev)
    for i, (s, c) in enumerate(zip(start, new)):
        at = torch.arange(s + c, device=dev)
        used[table[i].to(dev).long()[at // page], at % page] = True
    keys[(~used)[:, None].expand(-1, kv_heads, -1)] = float("nan")
    values.transpose(2, 3)[(~used)[:, None].expand(-1, kv_heads, -1)] = float("inf")
    assert torch.equal(paged_attention(q, keys, values, step, d ** -0.5), want)
    if new[0] > 2:
        # The last token of the first request: only its own row sees it.
        p = start[0] + new[0] - 1
        pg, off = int(table[0, p // page]), p % page
        keys[pg, :, off, 3] = float("nan")
        values[pg, 0, 5, off], values[pg, 1, 7, off] = float("-inf"), float("nan")
        got = paged_attention(q, keys, values, step, d ** -0.5)
        r = new[0] - 1
        assert torch.equal(got[:r], want[:r]) and torch.equal(got[r + 1:], want[r + 1:])
        assert bool(got[r].isnan().all())


def test_infinite_values_reach_the_rows_that_see_them(dev):
    new, start, d = [40], [50], 64
    q, keys, values, table, step = cache_case(dev, new, start, 4, 2, d, 16, torch.float16, 9)
    for p in (3, 60, 89):
        values[int(table[0, p // 16]), 0, p % 64, p % 16] = float("inf")
    got = paged_attention(q, keys, values, step, d ** -0.5).view(40, 4, d)
    for p in (3, 60, 89):
        sees = torch.arange(40, device=dev) + 50 >= p
        assert bool((got[sees][:, :2, p % 64] == float("inf")).all())
        assert bool(got[~sees][:, :, p % 64].isfinite().all())
    assert bool(got[:, 2:].isfinite().all())


def test_extreme_scores(dev):
    """Scores far apart, and all equal; the maximum in the first, a middle or the last position."""
    d = 64
    for at in (0, 77, 299):
        q, keys, values, table, step = cache_case(dev, [1], [299], 2, 1, d, 16, torch.bfloat16, at)
        q.fill_(8.0)
        keys.fill_(-8.0)
        keys[int(table[0, at // 16]), 0, at % 16] = 8.0
        got = paged_attention(q, keys, values, step, 1.0)
        assert torch.equal(got[0, :d], values[int(table[0, at // 16]), 0, :, at % 16])
        keys.fill_(8.0)
        check_attention(paged_attention(q, keys, values, step, 1.0), q, keys, values, table, [299], [1], 1.0, torch.bfloat16)


@pytest.mark.parametrize("new,start", [([1], [70]), ([50], [70]), ([1], [1500])])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales_that_are_not_positive(dev, new, start, scale):
    q, keys, values, table, step = cache_case(dev, new, start, 4, 2, 64, 16, torch.bfloat16, 2)
    check_attention(paged_attention(q, keys, values, step, scale), q, keys, values, table, start, new, scale, torch.bfloat16)


def test_an_empty_step_is_refused(dev):
    state = PageState.new(2, 64, 8, 16, dev)
    step = PagedStep(state, 2, 1, 2, 1, 64)
    pool = torch.zeros(8, 1, 16, 64, device=dev).half()
    with pytest.raises(ValueError, match="page_tables fills it"):
        paged_attention(torch.zeros(2, 128, device=dev).half(), pool, pool.transpose(2, 3).contiguous(), step, 0.1)


def test_rows_behind_the_last_request_are_left(dev):
    q, keys, values, table, step = cache_case(dev, [3, 1], [0, 20], 4, 2, 64, 16, torch.float16, 3, extra_rows=30)
    out = torch.full_like(q, 7.0)
    assert paged_attention(q, keys, values, step, 0.125, out=out) is out
    assert bool((out[4:] == 7.0).all())
    check_attention(out, q, keys, values, table, [0, 20], [3, 1], 0.125, torch.float16)


@pytest.mark.parametrize("native", [True, False])
def test_given_outputs_are_written_in_place(dev, monkeypatch, native):
    """Autograd sees the write; what needs a gradient, or inference mode, is refused."""
    q, keys, values, table, step = cache_case(dev, [3, 1], [0, 20], 4, 2, 64, 16, torch.float16, 3)
    if not native:
        monkeypatch.setattr(_ffi, "calls", lambda: SimpleNamespace(paged_write=lambda *a: None, paged_attention=lambda *a: None))
    rows = q.shape[0]
    k = torch.randn(rows, 128, device=dev).half()
    cos = torch.randn(rows, 64, device=dev).half()
    for call in (lambda out: paged_attention(q, keys, values, step, 0.125, out=out),
                 lambda out: rotary_paged_write(q, k, k, cos, cos, keys, values, step.slots, out=out)):
        out = torch.ones_like(q)
        w = torch.ones_like(q, requires_grad=True)
        y = w * out
        assert call(out) is out
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        with pytest.raises(RuntimeError, match="no backward pass"):
            call(torch.ones_like(q, requires_grad=True))
        with torch.inference_mode():
            inside = torch.ones_like(q)
            call(inside)
        with pytest.raises(RuntimeError, match="inference mode"):
            call(inside)


def test_strided_rows_pages_and_outputs(dev):
    d, new, start = 64, [9, 1], [30, 70]
    q, keys, values, table, step = cache_case(dev, new, start, 4, 2, d, 16, torch.bfloat16, 4)
    want = paged_attention(q, keys, values, step, 0.125)
    wide = torch.zeros(q.shape[0], q.shape[1] + 24, device=dev).bfloat16()
    wide[:, 8:8 + q.shape[1]] = q
    layers = torch.zeros(keys.shape[0], 3, *keys.shape[1:], device=dev).bfloat16()  # pools of three layers, page by page
    vlayers = torch.zeros(values.shape[0], 3, *values.shape[1:], device=dev).bfloat16()
    layers[:, 1], vlayers[:, 1] = keys, values
    out = torch.zeros_like(wide)
    paged_attention(wide[:, 8:8 + q.shape[1]], layers[:, 1], vlayers[:, 1], step, 0.125, out=out[:, 16:16 + q.shape[1]])
    assert torch.equal(out[:, 16:16 + q.shape[1]], want)
    assert not out[:, :16].any() and not out[:, 16 + q.shape[1]:].any()
    wide[:, 1:1 + q.shape[1]] = q
    assert torch.equal(paged_attention(wide[:, 1:1 + q.shape[1]], keys, values, step, 0.125), want)  # not 16-byte aligned


def test_pages_outside_the_pool_give_nan_to_the_rows_that_need_them(dev):
    new, start, d, page = [6, 1], [30, 40], 64, 16
    q, keys, values, table, step = cache_case(dev, new, start, 4, 2, d, page, torch.bfloat16, 6)
    want = paged_attention(q, keys, values, step, 0.125)
    state = step.state
    for bad in (-1, keys.shape[0], 2 ** 31 - 1, -2 ** 31):
        state.table[0, 2] = bad     # positions 32 to 47: rows 2 and on of the first request
        got = paged_attention(q, keys, values, step, 0.125)
        assert torch.equal(got[:2], want[:2]) and bool(got[2:6].isnan().all()) and torch.equal(got[6:], want[6:])


def test_a_pool_that_runs_short(dev):
    """The request that gets no page has NaN, the others their answer; the next call makes it good."""
    state = PageState.new(2, 64, 3, 16, dev)
    step = page_tables(state, i32([0, 0], dev), i32([30, 30], dev), rows=60, max_new=30, heads=2, kv_heads=1, head_dim=64)
    assert state.counts.tolist() == [0, 1] and state.held.tolist() == [2, 1]
    q = torch.randn(60, 128, device=dev).half()
    keys, values = torch.randn(3, 1, 16, 64, device=dev).half(), torch.randn(3, 1, 64, 16, device=dev).half()
    got = paged_attention(q, keys, values, step, 0.125)
    assert bool(got[:46].isfinite().all()) and bool(got[46:].isnan().all())
    page_tables(state, i32([0, 0], dev), i32([14, 30], dev), rows=60, max_new=30, step=None)
    assert state.counts.tolist() == [0, 0] and state.held.tolist() == [1, 2]


def test_large_pool_offsets_pass_32_bits(dev):
    """A pool of more than 2^31 elements: the last pages are read and written where they are."""
    d, page, kv = 128, 16, 8
    pages = 2 ** 31 // (kv * page * d) + 40
    keys = torch.zeros(pages, kv, page, d, dtype=torch.bfloat16, device=dev)
    values = torch.zeros(pages, kv, d, page, dtype=torch.bfloat16, device=dev)
    ids = [pages - 1, 0, pages - 2, 5]
    state = PageState(table=i32([ids], dev), held=i32([4], dev), free=i32([0] * pages, dev), counts=i32([0, 0], dev), page=page)
    step = page_tables(state, i32([0], dev), i32([50], dev), rows=50, max_new=50, heads=8, kv_heads=8, head_dim=d)
    g = torch.Generator(dev).manual_seed(1)
    q, k, v = (torch.randn(50, 1024, generator=g, device=dev).bfloat16() for _ in range(3))
    cos, sin = torch.ones(1, d, device=dev).bfloat16(), torch.zeros(1, d, device=dev).bfloat16()
    rotary_paged_write(q, k, v, cos, sin, keys, values, step.slots)
    assert torch.equal(keys[pages - 1, :, 3], k[3].view(8, d)) and torch.equal(values[pages - 2, :, :, 1], v[33].view(8, d))
    got = paged_attention(q, keys, values, step, d ** -0.5)
    check_attention(got, q, keys, values, torch.tensor([ids]), [0], [50], d ** -0.5, torch.bfloat16)


# ---------------------------------------------------------------- verification
def probabilities(g, shape, dtype, dev, std=2.0):
    return torch.softmax(torch.randn(*shape, generator=g, device=dev) * std, -1).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ks,vocab,certain", [
    ([4], 512, False), ([0, 1, 2, 3], 1, False), ([3, 0, 5], 4097, False), ([3, 1], 2049, False), ([2, 2], 4096, True), ([70, 64, 1], 777, False),
    ([4] * 20, 12289, False), ([1, 8, 0], 128256, True), ([2, 0, 3, 1], 290001, False),
])
def test_verify_drafts(dev, ks, vocab, certain, dtype):
    g = torch.Generator(dev).manual_seed(vocab + len(ks))
    n, most = len(ks), max(max(ks), 1)
    indptr = [0]
    for k in ks:
        indptr.append(indptr[-1] + k + 1)
    target = probabilities(g, (indptr[-1], vocab), dtype, dev)
    draft = probabilities(g, (n, most, vocab), dtype, dev)
    for i, k in enumerate(ks):  # drafts near the target's rows
        draft[i, :k] = (draft[i, :k].float() * 0.2 + target[indptr[i]:indptr[i] + k].float() * 0.8).to(dtype)
    tokens = draft.float().view(-1, vocab).multinomial(1, generator=g).view(n, most)
    accept, last = torch.rand(n, most, generator=g, device=dev), torch.rand(n, generator=g, device=dev)
    if certain:
        accept = accept * 0.01
    q = None if certain else draft
    got = verify_drafts(target, q, tokens, i32(indptr, dev), accept, last)
    want = ref.verify(target, q, tokens, indptr, accept, last)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.int64


def test_verify_edges(dev):
    """Ties, zeros, numbers at both ends, rows without mass, drafts outside the vocabulary, requests without rows."""
    v = 5000
    target = torch.zeros(9, v, device=dev)
    target[0, 4100] = 0.5
    target[0, 4999] = 0.5
    target[1, 7] = 1.0
    target[2, 10:20] = 0.1
    target[3] = float("nan")
    target[4] = 0.0
    target[5, 3] = 1.0
    target[6, 2], target[6, 4] = 0.25, 0.75
    target[7, 9] = 1.0
    target[8, 1], target[8, 4500] = 0.5, 0.5
    indptr = [0, 1, 2, 3, 4, 5, 5, 7, 9]
    n = 8
    draft = torch.zeros(n, 1, v, device=dev)
    draft[6, 0, 3] = 1.0        # equal to the target: nothing left at the rejection
    draft[7, 0, 9] = 0.5
    tokens = torch.zeros(n, 1, dtype=torch.int64, device=dev)
    tokens[6], tokens[7] = 3, v   # u * 1 < 1 fails only for u = 1; a token outside the vocabulary
    accept = torch.ones(n, 1, device=dev)
    for last in (0.0, 0.5, 1 - 2.0 ** -24, 1.0):
        w = torch.full((n,), last, device=dev)
        got = verify_drafts(target, draft, tokens, i32(indptr, dev), accept, w)
        want = ref.verify(target, draft, tokens, indptr, accept, w)
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1], last
    assert got[1][5].tolist() == [-1, -1] and got[1][3, 0] == -1 and got[1][4, 0] == -1


def test_verify_strided_and_empty(dev):
    g = torch.Generator(dev).manual_seed(3)
    target = probabilities(g, (6, 300), torch.float32, dev)
    steps = probabilities(g, (2, 3, 300), torch.float32, dev).transpose(0, 1)[:, :, :299]  # drafted step by step
    tokens = torch.randint(0, 299, (3, 5), generator=g, device=dev)[:, 1:3]
    accept, last = torch.rand(3, 4, generator=g, device=dev)[:, :2], torch.rand(3, generator=g, device=dev)
    indptr = [0, 3, 4, 6]
    got = verify_drafts(target[:, :299], steps, tokens, i32(indptr, dev), accept, last)
    want = ref.verify(target[:, :299], steps, tokens, indptr, accept, last)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    a, t = verify_drafts(target, None, torch.zeros(0, 2, dtype=torch.int64, device=dev), i32([0], dev),
                         torch.zeros(0, 2, device=dev), torch.zeros(0, device=dev))
    assert a.shape == (0,) and t.shape == (0, 3)
    a, t = verify_drafts(target, None, torch.zeros(6, 0, dtype=torch.int64, device=dev), i32(list(range(7)), dev),
                         torch.zeros(6, 0, device=dev), torch.rand(6, generator=g, device=dev))
    assert a.tolist() == [0] * 6 and t.shape == (6, 1)


# ---------------------------------------------------------------- together, captured
@pytest.mark.parametrize("longest", [600, 1600])  # without and with room for split ranges
def test_steps_captured_and_replayed(dev, longest):
    """Tables, write, attention and verification of a step in one graph, replayed with other lengths, equal the eager calls."""
    heads, kv_heads, d, page, n, most = 8, 2, 64, 16, 5, 3
    rows, vocab = n * (most + 1), 640
    g = torch.Generator(dev).manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g, device=dev).half()  # noqa: E731
    qkv = rn(rows, (heads + 2 * kv_heads) * d)
    q, k, v = qkv.split((heads * d, kv_heads * d, kv_heads * d), 1)
    cos, sin = rn(rows, d), rn(rows, d)
    target, draft = probabilities(g, (rows, vocab), torch.float32, dev), probabilities(g, (n, most, vocab), torch.float32, dev)
    tokens = torch.randint(0, vocab, (n, most), generator=g, device=dev)
    accept, last = torch.rand(n, most, generator=g, device=dev), torch.rand(n, generator=g, device=dev)
    start, new = i32([0] * n, dev), i32([4] * n, dev)

    def fresh():
        return (PageState.new(n, longest, 200, page, dev), torch.zeros(200, kv_heads, page, d, device=dev).half(),
                torch.zeros(200, kv_heads, d, page, device=dev).half())

    def make(state):
        return PagedStep(state, rows, most + 1, heads, kv_heads, d)

    def run(state, keys, values, step, out):
        page_tables(state, start, new, step=step)
        rot = rotary_paged_write(q, k, v, cos, sin, keys, values, step.slots)
        paged_attention(rot, keys, values, step, d ** -0.5, out=out)
        return verify_drafts(target, draft, tokens, step.row_indptr, accept, last)

    mine, theirs = fresh(), fresh()
    sa, sb = make(mine[0]), make(theirs[0])
    oa, ob = torch.zeros_like(q), torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*mine, sa, oa)
    torch.cuda.current_stream().wait_stream(side)
    page_tables(mine[0], i32([0] * n, dev), i32([0] * n, dev), rows=0, max_new=0)
    mine[1].zero_(), mine[2].zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = run(*mine, sa, oa)
    for lens in ([[0] * n, [4, 1, 2, 3, 4]], [[4, 1, 2, 3, 4], [1] * n], [[300, 2, 0, 4, 5], [4, 0, 4, 1, 2]],
                 [[0, 0, 590, 4, 5], [0, 1, 4, 4, 4]], [[longest - 10, 2, 0, 4, 5], [4, 0, 4, 1, 2]]):
        start.copy_(i32(lens[0], dev))
        new.copy_(i32(lens[1], dev))
        oa.fill_(3.0), ob.fill_(3.0)
        graph.replay()
        want = run(*theirs, sb, ob)
        torch.cuda.synchronize()
        for x, y in zip((oa, *mine[1:], sa.slots, sa.positions, mine[0].held, *res),
                        (ob, *theirs[1:], sb.slots, sb.positions, theirs[0].held, *want)):
            assert torch.equal(x, y)


def test_two_steps_of_one_state_on_two_streams(dev):
    """Attention over two steps' own plans and workspaces at once gives each one's own answer."""
    q1, keys, values, table, step1 = cache_case(dev, [1] * 4, [900, 2000, 300, 77], 8, 2, 128, 16, torch.bfloat16, 1)
    state = step1.state
    step2 = page_tables(state, i32([900, 2000, 300, 77], dev), i32([1] * 4, dev), rows=4, max_new=1, heads=8, kv_heads=2, head_dim=128)
    q2 = q1.flip(0).contiguous()
    want = paged_attention(q1, keys, values, step1, 0.1), paged_attention(q2, keys, values, step2, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            b = [paged_attention(q2, keys, values, step2, 0.1) for _ in range(8)]
        a = [paged_attention(q1, keys, values, step1, 0.1) for _ in range(8)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, want[0]) for x in a) and all(torch.equal(x, want[1]) for x in b)


@pytest.mark.parametrize("new,start,rows", [([1] * 4, [900, 2000, 300, 77], 4), ([300, 1, 7], [900, 2000, 0], 308)])
def test_a_step_that_was_only_recorded(dev, new, start, rows):
    """The launch that fills a step's work list stands in a graph that has not run: whatever the list's memory holds, the
    call keeps to its tensors.  Once the graph has run it answers."""
    q, keys, values, table, eager = cache_case(dev, new, start, 8, 2, 128, 16, torch.bfloat16, 1)
    want = paged_attention(q, keys, values, eager, 0.1)
    step = PagedStep(eager.state, rows, max(new), 8, 2, 128)
    first, more = i32(start, dev), i32(new, dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        page_tables(eager.state, first, more, step=step)
    out = torch.full_like(q, 7.0)
    for junk in (-1, 2 ** 31 - 1, -2 ** 31, 0, 1000, 1 << 24):
        step._ints.fill_(junk)
        paged_attention(q, keys, values, step, 0.1, out=out)
        assert bool((out == 7.0).all())
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(paged_attention(q, keys, values, step, 0.1), want)


@pytest.mark.parametrize("native", [True, False])
def test_what_torch_has_to_see_is_refused(dev, monkeypatch, native):
    """A launch past torch would drop a tangent, and a trace would keep its result as a constant."""
    q, keys, values, table, step = cache_case(dev, [3, 1], [0, 20], 4, 2, 64, 16, torch.float16, 3)
    k, cos = torch.randn(4, 128, device=dev).half(), torch.randn(4, 64, device=dev).half()
    target, tokens = probabilities(torch.Generator(dev).manual_seed(1), (4, 50), torch.float32, dev), torch.zeros(2, 1, dtype=torch.int64, device=dev)
    u, start, new, indptr = torch.zeros(2, 1, device=dev), i32([0, 20], dev), i32([3, 1], dev), i32([0, 2, 4], dev)
    if not native:
        none = lambda *a: None  # noqa: E731
        monkeypatch.setattr(_ffi, "calls", lambda: SimpleNamespace(page_tables=none, paged_write=none, paged_attention=none,
                                                                   verify_drafts=none))

    def attend(q, keys=keys, values=values):
        return paged_attention(q, keys, values, step, 0.125)

    def write(q, k=k, v=k, cos=cos):
        return rotary_paged_write(q, k, v, cos, cos, keys, values, step.slots)

    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: attend(dual(q)), lambda: attend(q, keys=dual(keys)), lambda: attend(q, values=dual(values)),
                     lambda: write(dual(q)), lambda: write(q, k=dual(k)), lambda: write(q, v=dual(k)), lambda: write(q, cos=dual(cos))):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
        got = attend(q)  # without a tangent
    assert torch.equal(got, attend(q))
    for f, x in ((lambda x: attend(x), q), (lambda x: write(x), q), (lambda p: verify_drafts(p, None, tokens, indptr, u, u[:, 0])[1], target),
                 (lambda c: page_tables(step.state, start, c, step=step).slots, new)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,), check_trace=False)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f)(x)
        f(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(attend)(q[None])
    with pytest.raises(RuntimeError):
        torch.func.jvp(attend, (q,), (q,))


@pytest.mark.parametrize("n", [5, 1200, 2100])  # one launch, and two
@pytest.mark.parametrize("rows", [0, 3, 15, 40])
def test_pages_go_to_the_tokens_that_the_rows_hold(dev, n, rows):
    """A request that gets fewer rows than it asked for takes pages for those only, and gives back the others."""
    start, new = [7, 20, 0, 0, 33] + [0] * (n - 5), [40, 12, 30, 60, 17] + [1] * (n - 5)
    state, sim = PageState.new(n, 64, 20 + n, 16, dev), ref.Pages(n, 4, 20 + n, 16)
    for starts, asked, room in (([0] * n, start, sum(start)), (start, new, rows), (start, [0] * n, 0), (start, new, rows + 9)):
        left, got = room, []
        for c in asked:
            got.append(min(c, left))
            left -= got[-1]
        step = page_tables(state, i32(starts, dev), i32(asked, dev), rows=room, max_new=60, heads=2, kv_heads=1, head_dim=64)
        check_step(state, sim, step, sim.step(starts, got, room), room)


def test_as_many_parts_as_a_step_can_have(dev):
    """Eight tiles of 64 parts each: the workspace has room for 512 parts of one key head's long tiles."""
    new, start = [16] * 8, [65520] * 8
    q, keys, values, table, step = cache_case(dev, new, start, 8, 1, 64, 256, torch.bfloat16, 5)
    assert step._c.workspace_bytes == (512 * 128 + 521 * 16) * 66 * 4
    check_attention(paged_attention(q, keys, values, step, 0.125), q, keys, values, table, start, new, 0.125, torch.bfloat16)


@pytest.mark.parametrize("rows", [0, 5])
def test_a_step_of_no_requests(dev, rows):
    state = PageState.new(0, 64, 4, 16, dev)
    none = i32([], dev)
    for heads in ({}, dict(heads=2, kv_heads=1, head_dim=64)):
        step = PagedStep(state, rows, 1, **heads)
        step._ints.fill_(77)
        state.counts[1] = 3
        page_tables(state, none, none, step=step)
        assert step.row_indptr.tolist() == [0] and step.positions.tolist() == [0] * rows and step.slots.tolist() == [-1] * rows
        assert state.counts.tolist() == [4, 0]
    out = torch.full((rows, 128), 7.0, device=dev).half()
    pool = torch.zeros(4, 1, 16, 64, device=dev).half()
    paged_attention(torch.zeros_like(out), pool, pool.view(4, 1, 64, 16), step, 0.1, out=out)
    assert bool((out == 7.0).all())


# ---------------------------------------------------------------- work lists of large steps (built by two launches)
def many_requests(seed, n):
    """Lengths of ``n`` requests: mostly short, some without tokens, long ranges and prompts among the first and the last."""
    rng = random.Random(seed)
    new = [rng.choice((0, 1, 1, 1, 3)) for _ in range(n)]
    start = [rng.randint(0, 60) for _ in range(n)]
    for i in (5, 700, n - 9):
        new[i], start[i] = 1, rng.randint(2500, 6000)
    for i in (17, n - 30):
        new[i], start[i] = rng.randint(100, 300), rng.randint(0, 3000)
    return new, start


LARGE = [
    # new, start, heads, kv_heads, d, page: more than 2048 rows, ranges of both kinds split
    ([1500, 1, 1, 700, 5, 0, 1], [4000, 9000, 3000, 0, 1200, 50, 0], 8, 2, 64, 16),
    ([2, 2100, 1, 40], [7000, 1100, 0, 2500], 16, 2, 128, 32),
    # more than 1024 requests: two and three rounds of the scan
    (*many_requests(1, 1300), 4, 1, 64, 16), (*many_requests(2, 2300), 2, 1, 128, 8),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", range(len(LARGE)))
def test_attention_of_large_steps(dev, case, dtype):
    new, start, heads, kv_heads, d, page = LARGE[case]
    assert sum(new) > 2048 or len(new) > 1024
    q, keys, values, table, step = cache_case(dev, new, start, heads, kv_heads, d, page, dtype, case)
    got = paged_attention(q, keys, values, step, d ** -0.5)
    check_attention(got, q, keys, values, table, start, new, d ** -0.5, dtype)


@pytest.mark.parametrize("seed", range(8))
def test_both_work_lists_of_one_step_agree(dev, seed):
    """One launch builds the list of a small step, two that of a step with room for many rows: the same items and parts,
    so the same results bit for bit."""
    rng = random.Random(seed)
    heads, kv_heads, d = rng.choice(((32, 8, 128), (4, 1, 64), (12, 2, 64), (8, 8, 128)))
    n = (1, 3, 30, 200, 900, 1024, 40, 9)[seed]
    new = [rng.choice((0, 1, 1, 2)) if n > 100 else rng.choice((0, 1, 4, rng.randint(5, 1200 // n + 5))) for _ in range(n)]
    new[0] = max(new[0], 1)
    start = [rng.choice((0, rng.randint(0, 100), rng.randint(0, 100), rng.randint(0, 3000 if n < 100 else 200))) for _ in range(n)]
    start[-1] = 4000
    q, keys, values, table, step = cache_case(dev, new, start, heads, kv_heads, d, 16, torch.bfloat16, seed)
    rows = sum(new)
    assert rows <= 2048
    roomy = page_tables(step.state, i32(start, dev), i32(new, dev), rows=2500, max_new=max(new), heads=heads, kv_heads=kv_heads,
                        head_dim=d)
    assert torch.equal(roomy.slots[:rows], step.slots) and torch.equal(roomy.row_indptr, step.row_indptr)
    wide = torch.cat((q, torch.zeros(2500 - rows, heads * d, dtype=q.dtype, device=dev)))
    assert torch.equal(paged_attention(wide, keys, values, roomy, d ** -0.5)[:rows], paged_attention(q, keys, values, step, d ** -0.5))
