"""The decoder over the paged cache (GPU): ragged prompts, decoding, chunks, captured steps and verified drafts give what
the same tokens give without a cache, each request with its own adapter."""

import pytest
import torch

from multi_lora_amd import AdapterWeights, MultiLoRAManager
from multi_lora_amd.decoder import Decoder, DecoderConfig, PagedKV
from multi_lora_amd.graph_decode import capture_graph
from multi_lora_amd.paged_decode import PagedDecode

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
