"""The decoder over the paged cache (GPU): ragged prompts, decoding, chunks, captured steps and verified drafts give what
the same tokens give without a cache, each request with its own adapter."""

import pytest
import torch

from multi_lora_amd import AdapterWeights, MultiLoRAManager
from multi_lora_amd.decoder import Decoder, DecoderConfig, PagedKV
from multi_lora_amd.graph_decode import capture_graph
from multi_lora_amd.paged_decode import PagedDecode

from tests import paged_ref as ref

pytestmark = pytest.mark.gpu

PROJ = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj",
        "mlp.down_proj")
NAMES = ["a", None, "b", "a"]
LENS = [5, 33, 1, 70]
# Logits of a two-layer bf16 model whose roundings differ along the way (the tolerance its other paths are held to).
ATOL = 6e-2


def build(dtype=torch.bfloat16):
    torch.manual_seed(0)
    cfg = DecoderConfig()
    model = Decoder(cfg).to("cuda", dtype).eval()
    adapters = {}
    for j, name in enumerate(("a", "b")):
        g = torch.Generator().manual_seed(10 + j)
        mods = {}
        for layer in range(cfg.num_hidden_layers):
            for p in PROJ:
                lin = model.get_submodule(f"layers.{layer}.{p}")
                mods[f"layers.{layer}.{p}"] = ((torch.randn(8, lin.in_features, generator=g) * 0.05).to(dtype),
                                               (torch.randn(lin.out_features, 8, generator=g) * 0.05).to(dtype))
        adapters[name] = AdapterWeights(rank=8, scaling=2.0, modules=mods)
    return MultiLoRAManager.from_adapters(model, adapters, max_loras_per_batch=4, max_lora_rank=16), cfg


def prompts(cfg, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab_size, (n,), generator=g).to("cuda") for n in LENS]


def whole(mgr, ids, name):
    """Logits of one sequence without a cache."""
    return mgr.forward_with_lora(input_ids=ids[None], lora_names=[name], seq_lens=[ids.numel()], use_cache=False).logits[0]


@torch.inference_mode()
def test_ragged_prompts_and_steps_equal_whole_sequences(dev):
    mgr, cfg = build()
    ps = prompts(cfg)
    step = PagedDecode.new(mgr, 4, 96)
    first = step.prefill(mgr, ps, NAMES)
    rows = torch.stack([whole(mgr, p, n)[-1] for p, n in zip(ps, NAMES)])
    top2 = rows.float().topk(2, -1).values
    clear = top2[:, 0] - top2[:, 1] > 2 * ATOL
    assert torch.equal(first[clear, 0], rows.argmax(-1)[clear])
    g = torch.Generator().manual_seed(8)
    seqs = list(ps)
    for _ in range(3):
        step.input_ids.copy_(torch.randint(0, cfg.vocab_size, (4, 1), generator=g))
        seqs = [torch.cat((s, t)) for s, t in zip(seqs, step.input_ids)]
        mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
        got = step.run(mgr).logits
        want = torch.stack([whole(mgr, s, n)[-1] for s, n in zip(seqs, NAMES)])
        torch.testing.assert_close(got.float(), want.float(), atol=ATOL, rtol=ATOL)
    assert step.lens.tolist() == [n + 3 for n in LENS]
    assert step.kv.state.held.tolist() == [-(-(n + 3) // 16) for n in LENS]


@torch.inference_mode()
def test_a_prompt_in_chunks_beside_decoding_requests(dev):
    """Continuous batching: request 3's prompt comes in two chunks while the others decode."""
    mgr, cfg = build()
    ps = prompts(cfg, 5)
    kv = PagedKV(cfg, 4, 96, dev, torch.bfloat16, page=8)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731

    def forward(start, new, ids, names):
        st = kv.tables(i32(*start), i32(*new), kv.new_step(sum(new) + 3, max(new)))
        live = [(n, c) for n, c in zip(names, new) if c]
        pad = torch.zeros(3, dtype=torch.long, device=dev)  # rows behind the last request's, of the base model
        return mgr.forward_with_lora(input_ids=torch.cat((ids, pad)), lora_names=[n for n, _ in live] + [None],
                                     seq_lens=[c for _, c in live] + [3], past_key_values=kv, paged_step=st).logits

    forward([0, 0, 0, 0], [5, 33, 1, 0], torch.cat(ps[:3]), NAMES)
    nxt = torch.randint(0, cfg.vocab_size, (3,), generator=torch.Generator().manual_seed(1)).to(dev)
    got = forward([5, 33, 1, 0], [1, 1, 1, 41], torch.cat((nxt, ps[3][:41])), NAMES)
    want = [whole(mgr, torch.cat((p, t[None])), n)[-1:] for p, t, n in zip(ps, nxt, NAMES)] + [whole(mgr, ps[3], NAMES[3])[:41]]
    torch.testing.assert_close(got[:44].float(), torch.cat(want).float(), atol=ATOL, rtol=ATOL)
    # request 1 leaves; request 3's second chunk
    got = forward([6, 0, 2, 41], [0, 0, 0, 29], ps[3][41:], NAMES)
    torch.testing.assert_close(got[:29].float(), whole(mgr, ps[3], NAMES[3])[41:].float(), atol=ATOL, rtol=ATOL)
    assert kv.state.held.tolist() == [1, 0, 1, 9]


@torch.inference_mode()
def test_captured_steps_equal_direct_ones(dev):
    mgr, cfg = build()
    ps = prompts(cfg, 6)
    recorded, direct = PagedDecode.new(mgr, 4, 96), PagedDecode.new(mgr, 4, 96)
    for s in (recorded, direct):
        s.input_ids.copy_(s.prefill(mgr, ps, NAMES))
    mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
    graph, out = capture_graph(mgr, recorded)
    assert recorded.lens.tolist() == LENS and recorded.kv.state.held.tolist() == [-(-n // 16) for n in LENS]
    for _ in range(6):
        graph.replay()
        want = direct.run(mgr).logits
        torch.cuda.synchronize()
        assert torch.equal(out.logits, want)
        nxt = want.argmax(-1, keepdim=True)
        recorded.input_ids.copy_(nxt)
        direct.input_ids.copy_(nxt)
    assert torch.equal(recorded.lens, direct.lens) and torch.equal(recorded.kv.state.held, direct.kv.state.held)


@torch.inference_mode()
def test_verified_drafts(dev):
    """Accepted drafts are kept as if they had been decoded, rejected ones leave nothing behind."""
    mgr, cfg = build()
    ps = prompts(cfg, 7)
    k = 3
    g = torch.Generator(dev).manual_seed(2)
    drafts = torch.randint(0, cfg.vocab_size, (4, k), generator=g, device=dev)
    start = torch.randint(0, cfg.vocab_size, (4, 1), generator=g, device=dev)
    last = torch.rand(4, generator=g, device=dev)
    step = PagedDecode.new(mgr, 4, 96)
    step.prefill(mgr, ps, NAMES)
    step.input_ids.copy_(start)
    mgr._setup_forward_batch(NAMES, seq_lens=[k + 1] * 4)
    # Certain drafts are accepted while u < p: u = 0 takes all, u = 1 none.
    u = torch.zeros(4, k, device=dev)
    u[1:3] = 1.0
    u[3, 1:] = 1.0
    accepted, tokens = step.verify(mgr, drafts, None, u, last)
    assert accepted.tolist() == [3, 0, 0, 1]
    assert step.lens.tolist() == [n + a + 1 for n, a in zip(LENS, (3, 0, 0, 1))]
    for i, a in enumerate(accepted.tolist()):
        assert tokens[i, :a].tolist() == drafts[i, :a].tolist() and tokens[i, a + 1:].tolist() == [-1] * (k - a)
        assert int(step.input_ids[i, 0]) == int(tokens[i, a])
        if a < k:
            assert int(tokens[i, a]) != int(drafts[i, a])  # a certain draft that was rejected has no mass left
    seqs = [torch.cat((p, s, d[:a], t)) for p, s, d, a, t in zip(ps, start, drafts, accepted.tolist(), step.input_ids)]
    mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
    got = step.run(mgr).logits
    want = torch.stack([whole(mgr, s, n)[-1] for s, n in zip(seqs, NAMES)])
    torch.testing.assert_close(got.float(), want.float(), atol=ATOL, rtol=ATOL)
    assert step.kv.state.held.tolist() == [-(-int(n) // 16) for n in step.lens.tolist()]
    assert step.kv.state.counts.tolist() == [4 * 6 - sum(step.kv.state.held.tolist()), 0]


def test_refusals(dev):
    mgr, cfg = build()
    step = PagedDecode.new(mgr, 2, 40)
    ids = torch.zeros(40, dtype=torch.long, device=dev)
    for bad in ([ids[:5]], [ids[:5], ids[:0]], [ids[:5], ids]):
        with pytest.raises(ValueError, match="prompts"):
            step.prefill(mgr, bad, ["a", "b"])
    fp32 = PagedKV(cfg, 2, 40, dev, torch.float32)
    with pytest.raises(ValueError, match="float16 or bfloat16"), torch.no_grad():
        Decoder(cfg).to(dev).forward_paged(ids[:2], fp32, fp32.tables(step.none, step.one, fp32.new_step(2, 1)))


# ---------------------------------------------------------------- tokens without a place
def short_of_pages():
    """A decoder's requests 0 (14 tokens) and 1 (15 tokens) on three pages of 16 positions."""
    mgr, cfg = build()
    g = torch.Generator().manual_seed(11)
    ps = [torch.randint(0, cfg.vocab_size, (n,), generator=g).to("cuda") for n in (14, 15)]
    step = PagedDecode.new(mgr, 2, 96, num_pages=3)
    step.input_ids.copy_(step.prefill(mgr, ps, ["a", "b"]))
    return mgr, cfg, step, [torch.cat((p, t)) for p, t in zip(ps, step.input_ids)]


def step_and_compare(mgr, step, seqs, names, live):
    """One token of every request: those in ``live`` equal their whole sequences, the others' rows are NaN."""
    mgr._setup_forward_batch(names, seq_lens=[1] * len(names))
    before = step.lens.tolist()
    got = step.run(mgr).logits
    for i, (s, n) in enumerate(zip(seqs, names)):
        if i in live:
            torch.testing.assert_close(got[i].float(), whole(mgr, s, n)[-1].float(), atol=ATOL, rtol=ATOL)
        else:
            assert bool(got[i].isnan().all())
    assert step.placed.tolist() == [int(i in live) for i in range(len(names))]
    assert step.lens.tolist() == [b + int(i in live) for i, b in enumerate(before)]


@torch.inference_mode()
def test_drafts_without_a_page_are_not_kept(dev):
    """Request 0 takes the last page and rejects its drafts; request 1's drafts have no place, and none of them counts as
    cached: what follows attends to its own tokens, not to what request 0 left in the page."""
    mgr, cfg, step, seqs = short_of_pages()
    g = torch.Generator(dev).manual_seed(2)
    drafts = torch.randint(0, cfg.vocab_size, (2, 3), generator=g, device=dev)
    u = torch.tensor([[1.0] * 3, [0.0] * 3], device=dev)
    mgr._setup_forward_batch(["a", "b"], seq_lens=[4, 4])
    accepted, tokens = step.verify(mgr, drafts, None, u, torch.rand(2, generator=g, device=dev))
    assert step.placed.tolist() == [4, 1] and accepted.tolist() == [0, 0] and step.lens.tolist() == [15, 16]
    assert tokens[:, 1:].tolist() == [[-1] * 3] * 2 and bool((tokens[:, 0] >= 0).all())
    assert torch.equal(step.input_ids, tokens[:, :1])
    seqs = [torch.cat((s, t)) for s, t in zip(seqs, step.input_ids)]
    for live in ((0, 1), (1,)):  # request 1 gets the page that request 0 gives back; then request 0 needs one
        step_and_compare(mgr, step, seqs, ["a", "b"], live)
        step.input_ids.copy_(torch.randint(0, cfg.vocab_size, (2, 1), generator=torch.Generator().manual_seed(len(live))))
        if 0 not in live:
            step.input_ids[0] = seqs[0][-1]
        seqs = [torch.cat((s, t)) if i in live else s for i, (s, t) in enumerate(zip(seqs, step.input_ids))]
        if len(live) == 2:
            assert step.lens.tolist() == [16, 17]
    # Verification of a request without any place: nothing accepted, nothing changed.
    before, ids = step.lens.tolist(), step.input_ids.clone()
    mgr._setup_forward_batch(["a", "b"], seq_lens=[4, 4])
    accepted, tokens = step.verify(mgr, drafts, None, torch.ones(2, 3, device=dev), torch.rand(2, generator=g, device=dev))
    assert step.placed.tolist() == [0, 4] and accepted.tolist() == [0, 0] and tokens[0].tolist() == [-1] * 4
    assert step.lens.tolist() == [before[0], before[1] + 1] and torch.equal(step.input_ids[0], ids[0])
    # Request 1 leaves: request 0 goes on where it was.
    step.lens[1] = 0
    seqs[1] = step.input_ids[1]
    step_and_compare(mgr, step, seqs, ["a", "b"], (0, 1))


@torch.inference_mode()
def test_the_last_positions_of_the_table(dev):
    """Drafts past the table's end are not looked at, and a full request stays as it is."""
    mgr, cfg = build()
    g = torch.Generator().manual_seed(4)
    ps = [torch.randint(0, cfg.vocab_size, (n,), generator=g).to("cuda") for n in (30, 7)]
    step = PagedDecode.new(mgr, 2, 32)
    step.input_ids.copy_(step.prefill(mgr, ps, ["a", "b"]))
    drafts = torch.randint(0, cfg.vocab_size, (2, 3), generator=g).to(dev)
    seqs = [torch.cat((p, t, d)) for p, t, d in zip(ps, step.input_ids, drafts)]
    mgr._setup_forward_batch(["a", "b"], seq_lens=[4, 4])
    accepted, tokens = step.verify(mgr, drafts, None, torch.zeros(2, 3, device=dev), torch.full((2,), 0.5, device=dev))
    assert step.placed.tolist() == [2, 4] and accepted.tolist() == [1, 3] and step.lens.tolist() == [32, 11]
    assert tokens[0, 0] == drafts[0, 0] and tokens[0, 1] >= 0 and tokens[0, 2:].tolist() == [-1, -1]
    # The token after the last draft that had a place is drawn from its row of the target.  Logits of at most 2 that are
    # off by ATOL (1 + 2) = 0.18 at most move a cumulated half to 1 / (1 + exp(-0.36)) = 0.59.
    p = torch.softmax(whole(mgr, seqs[0][:32], "a")[-1].double(), -1)
    before = p.cumsum(0)[tokens[0, 1]] - p[tokens[0, 1]]
    assert before - 0.1 < 0.5 < before + p[tokens[0, 1]] + 0.1
    seqs = [None, torch.cat((seqs[1], step.input_ids[1]))]
    for _ in range(2):
        lens = step.lens.tolist()
        mgr._setup_forward_batch(["a", "b"], seq_lens=[1, 1])
        got = step.run(mgr).logits
        assert bool(got[0].isnan().all()) and step.placed.tolist() == [0, 1] and step.lens.tolist() == [32, lens[1] + 1]
        torch.testing.assert_close(got[1].float(), whole(mgr, seqs[1], "b")[-1].float(), atol=ATOL, rtol=ATOL)
        seqs[1] = torch.cat((seqs[1], step.input_ids[1]))


@torch.inference_mode()
def test_prompts_that_the_pool_cannot_hold_are_refused(dev):
    mgr, cfg, step, _ = short_of_pages()
    lens, held = step.lens.tolist(), step.kv.state.held.tolist()
    ids = torch.zeros(40, dtype=torch.long, device=dev)
    with pytest.raises(ValueError, match="4 pages"):
        step.prefill(mgr, [ids, ids[:16]], ["a", "b"])
    assert step.lens.tolist() == lens and step.kv.state.held.tolist() == held
    step.prefill(mgr, [ids[:32], ids[:16]], ["a", "b"])
    assert step.kv.state.held.tolist() == [2, 1]


@torch.inference_mode()
def test_captured_steps_short_of_pages_equal_direct_ones(dev):
    mgr, cfg, direct, _ = short_of_pages()
    recorded = short_of_pages()[2]
    mgr._setup_forward_batch(["a", "b"], seq_lens=[1, 1])
    graph, out = capture_graph(mgr, recorded)
    for turn in range(6):
        graph.replay()
        want = direct.run(mgr).logits
        torch.cuda.synchronize()
        assert torch.equal(out.logits.isnan(), want.isnan())
        assert torch.equal(torch.nan_to_num(out.logits), torch.nan_to_num(want))
        assert torch.equal(recorded.lens, direct.lens) and torch.equal(recorded.placed, direct.placed)
        nxt = torch.where(direct.placed[:, None] > 0, want.argmax(-1, keepdim=True), direct.input_ids)
        recorded.input_ids.copy_(nxt)
        direct.input_ids.copy_(nxt)
    assert direct.lens.tolist() == [16, 21] and direct.placed.tolist() == [0, 1]


@torch.inference_mode()
def test_captured_verification_short_of_pages_equals_the_direct_one(dev):
    mgr, cfg, direct, _ = short_of_pages()
    recorded = short_of_pages()[2]
    g = torch.Generator(dev).manual_seed(3)
    drafts, u, last = torch.zeros(2, 3, dtype=torch.long, device=dev), torch.zeros(2, 3, device=dev), torch.zeros(2, device=dev)
    mgr._setup_forward_batch(["a", "b"], seq_lens=[4, 4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        recorded.verify(mgr, drafts, None, u, last)
        recorded.rewind()
    torch.cuda.current_stream().wait_stream(side)
    recorded.input_ids.copy_(direct.input_ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = recorded.verify(mgr, drafts, None, u, last)
    torch.cuda.current_stream().wait_stream(side)
    seen = set()
    for _ in range(8):
        drafts.random_(0, cfg.vocab_size, generator=g)
        u.copy_(torch.randint(0, 2, (2, 3), generator=g, device=dev))
        last.uniform_(generator=g)
        graph.replay()
        want = direct.verify(mgr, drafts, None, u, last)
        torch.cuda.synchronize()
        for x, y in zip((*res, recorded.lens, recorded.placed, recorded.input_ids),
                        (*want, direct.lens, direct.placed, direct.input_ids)):
            assert torch.equal(x, y)
        seen |= set(direct.placed.tolist())
    assert 0 in seen and 4 in seen and len(seen) > 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@torch.inference_mode()
def test_drawn_drafts(dev, dtype):
    """Drafts drawn from given probabilities, in steps between which requests decode: accepted as the definition says from
    the model's own probabilities, and what is kept gives the logits of the whole sequences."""
    mgr, cfg = build(dtype)
    ps = prompts(cfg, 9)
    k = 3
    g = torch.Generator(dev).manual_seed(6)
    step, twin = PagedDecode.new(mgr, 4, 112), PagedDecode.new(mgr, 4, 112)
    for s in (step, twin):
        s.input_ids.copy_(s.prefill(mgr, ps, NAMES))
    seqs = [torch.cat((p, t)) for p, t in zip(ps, step.input_ids)]
    kept = []
    for _ in range(3):
        q = torch.softmax(torch.randn(4, k, cfg.vocab_size, generator=g, device=dev) * 0.6, -1)
        drafts = q.view(-1, cfg.vocab_size).multinomial(1, generator=g).view(4, k)
        u, last = torch.rand(4, k, generator=g, device=dev), torch.rand(4, generator=g, device=dev)
        mgr._setup_forward_batch(NAMES, seq_lens=[k + 1] * 4)
        st = twin.kv.tables(twin.lens, torch.full_like(twin.lens, k + 1), twin.kv.new_step(4 * (k + 1), k + 1))
        logits = mgr.model(input_ids=torch.cat((twin.input_ids, drafts), 1), past_key_values=twin.kv, paged_step=st).logits
        want = ref.verify(torch.softmax(logits.float(), -1), q, drafts, st.row_indptr.tolist(), u, last)
        accepted, tokens = step.verify(mgr, drafts, q, u, last)
        assert accepted.tolist() == want[0] and tokens.tolist() == want[1] and step.placed.tolist() == [k + 1] * 4
        kept += want[0]
        seqs = [torch.cat((s, d[:a], t)) for s, d, a, t in zip(seqs, drafts, want[0], step.input_ids)]
        mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
        got = step.run(mgr).logits
        rows = torch.stack([whole(mgr, s, n)[-1] for s, n in zip(seqs, NAMES)])
        torch.testing.assert_close(got.float(), rows.float(), atol=ATOL, rtol=ATOL)
        step.input_ids.copy_(got.argmax(-1, keepdim=True))
        seqs = [torch.cat((s, t)) for s, t in zip(seqs, step.input_ids)]
        # The other decoder keeps the same tokens.
        twin.lens.copy_(step.lens - 1)
        twin.input_ids.copy_(torch.stack([s[-2:-1] for s in seqs]))
        mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
        assert torch.equal(twin.run(mgr).logits, got)
        twin.input_ids.copy_(step.input_ids)
    assert min(kept) < k and max(kept) > 0


@torch.inference_mode()
def test_ragged_float16_prompts_and_steps_equal_whole_sequences(dev):
    mgr, cfg = build(torch.float16)
    ps = prompts(cfg, 12)
    step = PagedDecode.new(mgr, 4, 96, page=32)
    step.input_ids.copy_(step.prefill(mgr, ps, NAMES))
    seqs = list(ps)
    for _ in range(3):
        seqs = [torch.cat((s, t)) for s, t in zip(seqs, step.input_ids)]
        mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
        got = step.run(mgr).logits
        want = torch.stack([whole(mgr, s, n)[-1] for s, n in zip(seqs, NAMES)])
        torch.testing.assert_close(got.float(), want.float(), atol=ATOL, rtol=ATOL)
        step.input_ids.copy_(got.argmax(-1, keepdim=True))
    assert step.placed.tolist() == [1] * 4


@torch.inference_mode()
def test_rewinding_after_a_request_has_left(dev):
    """Its prompt is no longer cached: it is not taken back to the prompt's end."""
    mgr, cfg, step, seqs = short_of_pages()
    step_and_compare(mgr, step, seqs, ["a", "b"], (0, 1))
    step.lens[1] = 0
    seqs[1] = step.input_ids[1].clone()
    step.input_ids[0] = 3
    step_and_compare(mgr, step, [torch.cat((seqs[0], step.input_ids[0])), seqs[1]], ["a", "b"], (0, 1))
    step.rewind()
    assert step.lens.tolist() == [14, 1] and step.kv.state.held.tolist() == [1, 1]
    step.input_ids.copy_(torch.tensor([[5], [6]]))
    seqs = [torch.cat((seqs[0][:14], step.input_ids[0])), torch.cat((seqs[1], step.input_ids[1]))]
    step_and_compare(mgr, step, seqs, ["a", "b"], (0, 1))


@torch.inference_mode()
def test_prompts_that_do_not_get_through_leave_an_empty_cache(dev):
    mgr, cfg, step, _ = short_of_pages()
    assert step.placed.tolist() == [14, 15]
    ids = torch.arange(20, dtype=torch.long, device=dev)
    with pytest.raises(ValueError):
        step.prefill(mgr, [ids, ids[:3]], ["a"])  # one name for two prompts
    assert step.lens.tolist() == [0, 0]
    step.rewind()
    assert step.lens.tolist() == [0, 0] and step.kv.state.counts.tolist() == [3, 0]
    step.input_ids.copy_(ids[4:6, None])
    step_and_compare(mgr, step, [ids[4:5], ids[5:6]], ["a", "b"], (0, 1))


@torch.inference_mode()
def test_fused_projections_over_the_paged_cache(dev, monkeypatch):
    """q, k and v as columns of one fused output."""
    monkeypatch.setenv("MULTI_LORA_FUSED_QKV", "all")
    monkeypatch.setenv("MULTI_LORA_FUSED_GATE_UP", "1")
    mgr, cfg = build()
    ps = prompts(cfg, 14)
    step = PagedDecode.new(mgr, 4, 96)
    step.input_ids.copy_(step.prefill(mgr, ps, NAMES))
    mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
    got = step.run(mgr).logits
    want = torch.stack([whole(mgr, torch.cat((p, t)), n)[-1] for p, t, n in zip(ps, step.input_ids, NAMES)])
    torch.testing.assert_close(got.float(), want.float(), atol=ATOL, rtol=ATOL)


@torch.inference_mode()
def test_verification_is_not_captured_before_its_first_call(dev):
    """What its step is made of would be filled by the graph alone, and an eager call before that read memory as it was."""
    mgr, cfg, step, _ = short_of_pages()
    other = short_of_pages()[2]
    drafts, u, last = torch.zeros(2, 2, dtype=torch.long, device=dev), torch.ones(2, 2, device=dev), torch.zeros(2, device=dev)
    stream = torch.cuda.Stream()
    mgr._setup_forward_batch(["a", "b"], seq_lens=[3, 3])
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other.verify(mgr, drafts, None, u, last)  # the adapters' workspace of the stream exists
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="once before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            step.verify(mgr, drafts, None, u, last)
    accepted, _ = step.verify(mgr, drafts, None, u, last)
    assert accepted.tolist() == [0, 0] and step.placed.tolist() == [3, 1] and step.lens.tolist() == [15, 16]
