"""What the paged cache's entry points refuse before anything is launched (CPU), and the bounds of a step's work list."""

import ctypes
import random

import pytest
import torch

from multi_lora_amd import _ffi
from multi_lora_amd.decoder import Decoder, DecoderConfig, PagedKV, StaticKV
from multi_lora_amd.kernels import PagedStep, PageState, page_tables, paged_attention, rotary_paged_write, verify_drafts
from tests import paged_ref as ref

BF, F16, F32 = _ffi.MLORA_BF16, _ffi.MLORA_F16, _ffi.MLORA_F32


def pages(**kw):
    d = dict(table=4096, table_stride=8, held=8192, free=12288, counts=16384, n=4, width=8, num_pages=32, page=16)
    d.update(kw)
    return _ffi.Pages(*[d[f] for f, _ in _ffi.Pages._fields_])


def step(**kw):
    d = dict(row_indptr=1 << 20, kv_lens=2 << 20, positions=3 << 20, slots=4 << 20, plan=5 << 20, workspace=6 << 20,
             plan_bytes=1 << 30, workspace_bytes=1 << 40, rows=9, max_new=4)
    d.update(kw)
    return _ffi.PagedStep(*[d[f] for f, _ in _ffi.PagedStep._fields_])


def said(text):
    return text in _ffi.lib().mlora_last_error().decode()


def test_page_tables_arguments():
    def call(p=None, s=None, start=64, new=128, heads=8, kv=2, d=64, scratch=256):
        return _ffi.lib().mlora_page_tables(ctypes.byref(p or pages()), start, new, ctypes.byref(s or step()), heads, kv, d,
                                            scratch, None)

    for page in (0, 4, 12, 2048, -16):
        assert call(pages(page=page)) == -2 and said("power of two")
    assert call(pages(n=-1)) == -1 and call(pages(width=-1)) == -1 and call(pages(num_pages=-1)) == -1
    assert call(pages(num_pages=1 << 28)) == -2 and said("2^31")
    assert call(pages(n=1 << 20, width=1 << 12, table_stride=1 << 12)) == -2 and said("2^31")
    assert call(pages(table_stride=7)) == -1 and said("table row stride")
    assert call(s=step(rows=-1)) == -1 and call(s=step(rows=(1 << 20) + 1)) == -2 and said("2^20")
    assert call(d=96) == -2 and call(heads=7) == -2 and call(kv=0) == -2 and call(heads=2048) == -2
    assert call(s=step(plan_bytes=16)) == -3 and said("plan of 16 bytes")
    for field in ("table", "held", "free", "counts"):
        assert call(pages(**{field: None})) == -1 and said("null")
    for field in ("row_indptr", "kv_lens", "positions", "slots"):
        assert call(s=step(**{field: None})) == -1 and said("null")
    assert call(start=None) == -1 and call(new=None) == -1 and call(scratch=None) == -1
    assert _ffi.lib().mlora_page_tables(None, 64, 128, ctypes.byref(step()), 8, 2, 64, 256, None) == -1
    assert _ffi.lib().mlora_page_tables(ctypes.byref(pages()), 64, 128, None, 8, 2, 64, 256, None) == -1


def test_write_arguments():
    def call(q=1 << 12, qs=512, ks=128, vs=128, rs=64, rot=BF, rows=3, heads=8, kv=2, d=64, keys=1 << 20, kps=2 * 64 * 16,
             vps=2 * 64 * 16, n=10, page=16, qo=1 << 13, qos=512, dt=BF, slots=64):
        return _ffi.lib().mlora_rotary_paged_write(q, qs, 1 << 14, ks, 1 << 15, vs, 1 << 16, 1 << 17, rs, rot, slots, rows,
                                                   heads, kv, d, keys, kps, 1 << 21, vps, n, page, qo, qos, dt, None)

    assert call(dt=F32) == -2 and call(rot=F16) == -2 and call(d=32) == -2 and call(page=24) == -2
    assert call(rows=-1) == -1 and call(heads=0) == -1 and call(kv=0) == -1
    for kw in (dict(qs=511), dict(ks=127), dict(vs=127), dict(rs=-1), dict(kps=2047), dict(vps=2047), dict(qos=511)):
        assert call(**kw) == -1 and said("strides"), kw
    for kw in (dict(q=None), dict(keys=None), dict(qo=None), dict(slots=None)):
        assert call(**kw) == -1 and said("null"), kw
    assert call(rows=0) == 0


def test_attention_arguments():
    def call(q=1 << 12, qs=512, keys=1 << 20, kps=2048, vps=2048, p=None, s=None, out=1 << 13, os_=512, heads=8, kv=2, d=64,
             dt=BF):
        return _ffi.lib().mlora_paged_attention(q, qs, keys, kps, 1 << 21, vps, ctypes.byref(p or pages()),
                                                ctypes.byref(s or step()), out, os_, heads, kv, d, 0.125, dt, None)

    assert call(dt=F32) == -2 and call(d=80) == -2 and call(heads=9) == -2 and call(p=pages(page=9)) == -2
    for kw in (dict(qs=511), dict(os_=511), dict(kps=2047), dict(vps=2047)):
        assert call(**kw) == -1 and said("strides"), kw
    for kw in (dict(q=1 << 12 | 2), dict(qs=516), dict(os_=516), dict(out=(1 << 13) + 8), dict(kps=2052), dict(keys=(1 << 20) + 8)):
        assert call(**kw) == -2 and said("aligned"), kw
    for kw in (dict(q=None), dict(keys=None), dict(out=None), dict(s=step(plan=None)), dict(p=pages(table=None)),
               dict(s=step(row_indptr=None)), dict(s=step(kv_lens=None))):
        assert call(**kw) == -1 and said("null"), kw
    assert call(s=step(plan_bytes=8)) == -3
    long_table = pages(width=4096, table_stride=4096)
    assert call(p=long_table, s=step(workspace_bytes=8)) == -3 and call(p=long_table, s=step(workspace=None)) == -3
    assert call(p=pages(num_pages=0)) == -1 and said("without pages")
    assert call(s=step(rows=0)) == 0 and call(p=pages(n=0)) == 0


def test_verify_arguments():
    lib = _ffi.lib()
    need = lib.mlora_verify_workspace_bytes(3, 5000)
    assert need == 3 * 3 * 2 * 8 and lib.mlora_verify_workspace_bytes(3, 0) == 0

    def call(target=1 << 12, ts=5000, rows=9, draft=1 << 20, s0=20000, tokens=1 << 13, accept=1 << 14, last=64, n=3, most=4,
             vocab=5000, ws=1 << 22, bytes_=need, dt=F32, indptr=32):
        return lib.mlora_verify_drafts(target, ts, rows, draft, s0, 5000, tokens, 4, indptr, accept, 4, last, n, most, vocab,
                                       128, 256, dt, ws, bytes_, None)

    assert call(dt=5) == -1 and call(n=-1) == -1 and call(most=-1) == -1 and call(vocab=0) == -1 and call(rows=-1) == -1
    assert call(ts=4999) == -1 and call(s0=-1) == -1 and call(vocab=(1 << 28) + 1, ts=1 << 30) == -2
    for kw in (dict(target=None), dict(tokens=None), dict(accept=None), dict(last=None), dict(indptr=None)):
        assert call(**kw) == -1 and said("null"), kw
    assert call(ws=None) == -3 and call(bytes_=need - 1) == -3
    assert call(n=0) == 0


def test_python_checks():
    st = PageState.new(3, 50, 10, 16, "cpu")
    assert st.table.shape == (3, 4) and st.counts.tolist() == [10, 0] and st.free.tolist() == list(range(9, -1, -1))
    lens = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        page_tables(st, lens, lens, rows=1, max_new=1)
    with pytest.raises(ValueError, match="power of two"):
        PageState.new(3, 50, 10, 12, "cpu")
    with pytest.raises(ValueError, match="held"):
        PageState(table=st.table, held=st.held[:2], free=st.free, counts=st.counts, page=16)
    with pytest.raises(ValueError, match="table"):
        PageState(table=st.table.t(), held=st.held, free=st.free, counts=st.counts, page=16)
    with pytest.raises(ValueError, match="counts"):
        PageState(table=st.table, held=st.held, free=st.free, counts=st.counts.long(), page=16)
    with pytest.raises(ValueError, match="together"):
        PagedStep(st, 4, 4, heads=8)
    with pytest.raises(ValueError, match="rows"):
        PagedStep(st, -1, 4)
    with pytest.raises(ValueError, match="head_dim"):
        PagedStep(st, 4, 4, heads=8, kv_heads=2, head_dim=80)
    s = PagedStep(st, 4, 4, heads=8, kv_heads=2, head_dim=64)
    q = torch.zeros(4, 512, dtype=torch.bfloat16)
    keys, values = torch.zeros(10, 2, 16, 64).bfloat16(), torch.zeros(10, 2, 64, 16).bfloat16()
    with pytest.raises(ValueError, match="page_tables fills it"):
        paged_attention(q, keys, values, s, 0.125)
    s.filled = True
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attention(q, keys, values, s, 0.125)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        rotary_paged_write(q, q[:, :128], q[:, :128], q[:, :64], q[:, :64], keys, values, lens)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        verify_drafts(torch.ones(1, 8), None, torch.zeros(1, 1, dtype=torch.int64), lens[:2], torch.ones(1, 1), torch.ones(1))


def test_the_plain_allocator_itself():
    """The allocator that the GPU tests compare with: no page is held twice or lost, and giving back restores the stack."""
    rng = random.Random(2)
    sim = ref.Pages(6, 10, 40, 8)
    lens = [0] * 6
    for _ in range(60):
        start = [rng.choice((0, l, max(0, l - 3))) for l in lens]
        new = [rng.randint(0, 80 - s) if rng.random() < 0.4 else 0 for s in start]
        before, had = list(sim.stack), list(sim.held)
        sim.step(start, new, sum(new))
        held = [p for i in range(6) for p in sim.table[i][:sim.held[i]]]
        assert sorted(held + sim.stack) == list(range(40))
        if all(h >= b for h, b in zip(sim.held, had)):
            again = [b * 8 for b in had]
            sim.step(again, [0] * 6, 0)
            assert sim.stack == before and sim.held == had
        lens = [h * 8 for h in sim.held]


def test_decoder_arguments():
    """What a paged step does not follow is refused, not ignored."""
    cfg = DecoderConfig()
    model, ids = Decoder(cfg), torch.zeros(1, 4, dtype=torch.long)
    kv, other = PagedKV(cfg, 2, 40, "cpu", torch.float32), PagedKV(cfg, 2, 40, "cpu", torch.float32)
    step = kv.new_step(4, 4)

    def call(**kw):
        return model(input_ids=ids, **{"past_key_values": kv, "paged_step": step, **kw})

    with pytest.raises(ValueError, match="its tables filled"):
        call()
    step.filled = True
    for kw in (dict(attention_mask=torch.ones(1, 4)), dict(position_ids=torch.zeros(1, 4, dtype=torch.long)),
               dict(cache_position=torch.arange(4)), dict(use_cache=False)):
        with pytest.raises(ValueError, match="no attention_mask"):
            call(**kw)
    for kw in (dict(paged_step=None), dict(past_key_values=other), dict(paged_step=PagedStep(kv.state, 4, 4))):
        with pytest.raises(ValueError, match="needs the paged_step"):
            call(**kw)
    with pytest.raises(ValueError, match="4 packed token ids"):
        model(input_ids=ids[:, :3], past_key_values=kv, paged_step=step)
    with pytest.raises(RuntimeError, match="no CPU fallback"), torch.no_grad():
        call()
    for kw in (dict(), dict(past_key_values=StaticKV(cfg, 1, 8, "cpu", torch.float32))):
        with pytest.raises(ValueError, match="go with a PagedKV"):
            model(input_ids=ids, paged_step=step, **kw)
        with pytest.raises(ValueError, match="go with a PagedKV"):
            model(input_ids=ids, logit_rows=torch.tensor([1]), **kw)


CUS = 256                      # without a GPU the library counts these
SPLIT_FROM = (256 + 384, 1024)  # longest range that no step splits, short and long


def slot_caps(n, rows, max_new, max_kv, heads, kv_heads):
    """(rows a tile, parts of split ranges that the workspace holds) of both kinds of a step's work items."""
    rep, target = heads // kv_heads, 2 * CUS
    most, every = min(max_new, rows) * rep, rows * rep
    bm = 32 if 16 < most <= 32 else 16
    caps = []
    for k, tile, tiles in ((0, bm, min(n, rows)), (1, 128, every // 128 + min(n, every // (bm + 1)) if most > bm else 0)):
        extra = target // kv_heads + 1 if tiles and max_kv > SPLIT_FROM[k] else 0
        caps.append((tile, min(tiles + extra, (1 if k else 2) * target // kv_heads) if extra else 0))
    return caps


@pytest.mark.parametrize("seed", range(6))
def test_a_steps_workspace_holds_the_parts_of_any_lengths(seed):
    """The workspace has room for every part that the split rule can make of a step's ranges, and for little more."""
    rng = random.Random(seed)
    full = 0.0
    for _ in range(400):
        kv_heads = rng.choice((1, 2, 4, 8, 32, 600))
        rep = rng.choice((1, 4, 7, 8, 16)) if kv_heads < 600 else 1
        d, n, page = rng.choice((64, 128)), rng.choice((1, 3, 20, 300)), 16
        new = [rng.choice((1, 1, 5, rng.randint(1, 3000))) for _ in range(n)]
        lens = [c + (0 if rng.random() < 0.1 else rng.choice((rng.randint(0, 500), 2048, 65536 - c % 4, rng.randint(0, 200000)))) for c in new]
        if rng.random() < 0.3:
            new, lens = [16] * n, [65536] * n
        max_kv = -(-max(lens) // page) * page
        caps = slot_caps(n, sum(new), max(new), max_kv, kv_heads * rep, kv_heads)
        plan, ws = ctypes.c_size_t(), ctypes.c_size_t()
        assert _ffi.lib().mlora_paged_step_bytes(n, sum(new), max(new), max_kv, kv_heads * rep, kv_heads, d, ctypes.byref(plan),
                                                 ctypes.byref(ws)) == 0
        assert ws.value == sum(slots * kv_heads * tile * (d + 2) * 4 for tile, slots in caps)
        # The split rule, on exact numbers: the least length of a part, and the parts of each tile.
        tiles = [[], []]
        for c, length in zip(new, lens):
            k = c * rep > caps[0][0]
            tiles[k] += [length] * (-(-c * rep // caps[k][0]))
        for k in (0, 1):
            split = -(-max(-(-sum(tiles[k]) * kv_heads // (2 * CUS)), (256, 1024)[k]) // 64) * 64
            if len(tiles[k]) * kv_heads >= 4 * 2 * CUS:
                continue
            parts = [max(length // split, 1) if k else -(-length // split) for length in tiles[k]]
            if k == 0 and max(tiles[0], default=0) - 384 <= split:
                continue
            used = sum(p for p in parts if p > 1)
            assert used <= caps[k][1]
            full = max(full, used / max(caps[k][1], 1))
    assert full == 1.0
