"""A model served in 8 bits (GPU): int8 projections beneath 16-bit adapters and the 8-bit paged cache, together, against
the same model with both computed plainly from their definitions."""

import copy

import pytest
import torch
import torch.nn as nn

from multi_lora_amd import Int8Linear, MultiLoRAManager, decoder, quantize_base
from multi_lora_amd.graph_decode import DecodeStep, capture_graph
from multi_lora_amd.kernels import Int8Rows
from multi_lora_amd.layers import LinearWithLoRA
from multi_lora_amd.paged_decode import PagedDecode

from tests import fp8_ref
from tests import paged_ref as ref
from tests.int8_ref import codes_of
from tests.test_gpu_paged_decode import ATOL, LENS, NAMES, build, prompts

pytestmark = pytest.mark.gpu


class PlainInt8(nn.Module):
    """An Int8Linear computed from its definition in 64 bits."""

    def __init__(self, layer: Int8Linear) -> None:
        super().__init__()
        self.w = layer.weight.to_rows().double() * layer.weight.scales.double()[:, None]
        self.bias = None

    def forward(self, x):
        codes, scales = (t.to(x.device) for t in codes_of(x.reshape(-1, x.shape[-1])))
        y = (codes * scales[:, None]) @ self.w.t()
        return y.to(x.dtype).view(*x.shape[:-1], -1)


def plain_write(q, k, v, cos, sin, pool, step, out=None):
    d, rows = pool.shape[3], step.rows
    turn = lambda x: (x.double().view(rows, -1, d) * cos.double() + x.double().view(rows, -1, d).roll(d // 2, -1) * sin.double())  # noqa: E731
    held = [t.view(torch.uint8).cpu() for t in (pool.keys, pool.values)] + [pool.key_scales.cpu(), pool.value_scales.cpu()]
    fp8_ref.write(*held, turn(k).cpu(), v.double().cpu().view(rows, -1, d), step.slots.tolist(), pool.dtype)
    for to, t in zip((pool.keys.view(torch.uint8), pool.values.view(torch.uint8), pool.key_scales, pool.value_scales), held):
        to.copy_(t)
    return turn(q).to(q.dtype).view(rows, -1)


def plain_attention(q, pool, step, scale, out=None):
    lens, indptr = step.kv_lens.tolist(), step.row_indptr.tolist()
    new = [b - a for a, b in zip(indptr, indptr[1:])]
    keys, values = pool.dequantize()
    used = indptr[-1]
    y, _ = ref.attention(q[:used], keys, values, step.state.table.cpu(), [l - c for l, c in zip(lens, new)], new, scale)
    return torch.cat((y.to(q.dtype), torch.zeros_like(q[used:])))


def quantised(dtype=torch.bfloat16):
    mgr, cfg = build(dtype)
    assert quantize_base(mgr.model) == 7 * cfg.num_hidden_layers
    assert isinstance(mgr.model.lm_head, nn.Linear)
    assert all(isinstance(w.base_layer, Int8Linear) for w in mgr.lora_wrappers.values())
    return mgr, cfg


def plainly(mgr):
    """The manager's wrappers over the definition."""
    for w in mgr.lora_wrappers.values():
        w.base_layer = PlainInt8(w.base_layer)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@torch.inference_mode()
def test_prompts_steps_and_drafts_together(dev, monkeypatch, dtype):
    """Ragged prompts, decoding and verified drafts with every request's adapter."""
    mgr, cfg = quantised(dtype)
    ps = prompts(cfg, 4)
    g = torch.Generator().manual_seed(8)
    nexts = [torch.randint(0, cfg.vocab_size, (4, 1), generator=g).to(dev) for _ in range(3)]
    drafts = torch.randint(0, cfg.vocab_size, (4, 3), generator=g).to(dev)
    u = torch.tensor([[0., 0., 0.], [1., 0., 0.], [0., 1., 0.], [0., 0., 1.]], device=dev)

    def run():
        step = PagedDecode.new(mgr, 4, 96, fp8=True)
        step.prefill(mgr, ps, NAMES)
        logits = []
        for ids in nexts:
            step.input_ids.copy_(ids)
            mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
            logits.append(step.run(mgr).logits.float())
        step.input_ids.copy_(nexts[0])
        mgr._setup_forward_batch(NAMES, seq_lens=[4] * 4)
        accepted, _ = step.verify(mgr, drafts, None, u, torch.full((4,), 0.5, device=dev))
        step.input_ids.copy_(nexts[1])
        mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
        logits.append(step.run(mgr).logits.float())
        return torch.cat(logits), accepted, step

    got, accepted, step = run()
    again, *_ = run()
    assert torch.equal(got, again)
    assert accepted.tolist() == [3, 0, 1, 2]
    assert step.lens.tolist() == [n + 5 + a for n, a in zip(LENS, accepted.tolist())]
    assert step.kv.pools[0].keys.dtype == torch.float8_e4m3fn
    plainly(mgr)
    monkeypatch.setattr(decoder, "rotary_paged_write_fp8", plain_write)
    monkeypatch.setattr(decoder, "paged_attention_fp8", plain_attention)
    want, *_ = run()
    torch.testing.assert_close(got, want, atol=ATOL, rtol=ATOL)


@torch.inference_mode()
def test_captured_steps_equal_direct_ones(dev):
    mgr, cfg = quantised()
    ps = prompts(cfg, 6)
    recorded, direct = PagedDecode.new(mgr, 4, 96, fp8=True), PagedDecode.new(mgr, 4, 96, fp8=True)
    for s in (recorded, direct):
        s.input_ids.copy_(s.prefill(mgr, ps, NAMES))
    mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
    graph, out = capture_graph(mgr, recorded)
    # The warm-up's tokens are still in the blocks' exponents, which only grow: the direct steps have them too.
    for _ in range(3):
        direct.run(mgr)
    direct.rewind()
    for _ in range(6):
        graph.replay()
        want = direct.run(mgr).logits
        torch.cuda.synchronize()
        assert torch.equal(out.logits, want)
        nxt = want.argmax(-1, keepdim=True)
        recorded.input_ids.copy_(nxt)
        direct.input_ids.copy_(nxt)


@torch.inference_mode()
def test_a_static_cache_over_int8_projections(dev):
    """The decode step of equal lengths, captured, and prompts: the same projections."""
    mgr, cfg = quantised()
    ids = torch.randint(0, cfg.vocab_size, (4, 20), generator=torch.Generator().manual_seed(1)).to(dev)
    step = DecodeStep.new(mgr, 4, 20, 40)
    step.input_ids.copy_(step.prefill(mgr, ids, torch.ones_like(ids), NAMES))
    token = step.input_ids.clone()
    mgr._setup_forward_batch(NAMES, seq_lens=[1] * 4)
    graph, out = capture_graph(mgr, step)
    graph.replay()
    torch.cuda.synchronize()
    got = out.logits[:, -1].float().clone()
    plainly(mgr)
    want = mgr.forward_with_lora(input_ids=torch.cat((ids, token), 1), lora_names=NAMES, seq_lens=[21] * 4, use_cache=False).logits
    torch.testing.assert_close(got, want[:, -1].float(), atol=ATOL, rtol=ATOL)


@torch.inference_mode()
def test_fused_projections(dev, monkeypatch):
    """q|k|v and gate|up as one product each: the groups' base products are those of their parts, bit for bit."""
    monkeypatch.setenv("MULTI_LORA_FUSED_QKV", "all")
    monkeypatch.setenv("MULTI_LORA_FUSED_GATE_UP", "1")
    mgr, cfg = build()
    with pytest.raises(RuntimeError, match="fused group"):
        quantize_base(mgr.model)
    torch.manual_seed(0)
    model = decoder.Decoder(cfg).to("cuda", torch.bfloat16).eval()
    quantize_base(model)
    store = mgr._weight_store
    apart = {n: m for n, m in model.named_modules() if isinstance(m, Int8Linear)}
    weights = {n: m.weight for n, m in apart.items()}
    fused = MultiLoRAManager.from_adapters(model, store, max_loras_per_batch=4, max_lora_rank=16)
    for name, w in fused.lora_wrappers.items():
        x = torch.randn(5, 1, w.base_layer.in_features, device=dev).bfloat16()
        assert torch.equal(w.base_layer.weight.to_rows(), weights[name].to_rows())
        if w.qkv_group is not None:
            a, b = w.qkv_slice
            assert torch.equal(w.qkv_group._base(x)[..., a:b], w.base_layer(x))
            assert w.base_layer.weight.codes.data_ptr() == w.qkv_group.weight.codes[:, a // 16:].data_ptr()  # a view
    ids = torch.randint(0, cfg.vocab_size, (1, 33), generator=torch.Generator().manual_seed(1)).to(dev)
    got = fused.forward_with_lora(input_ids=ids, lora_names=["a"], seq_lens=[33], use_cache=False).logits
    monkeypatch.setenv("MULTI_LORA_FUSED_QKV", "0")
    monkeypatch.setenv("MULTI_LORA_FUSED_GATE_UP", "0")
    single, _ = quantised()
    want = single.forward_with_lora(input_ids=ids, lora_names=["a"], seq_lens=[33], use_cache=False).logits
    torch.testing.assert_close(got.float(), want.float(), atol=ATOL, rtol=ATOL)


def test_the_module(dev):
    torch.manual_seed(1)
    lin = nn.Linear(100, 37, device=dev, dtype=torch.bfloat16)
    layer = Int8Linear.from_linear(lin)
    x = torch.randn(3, 5, 100, device=dev, dtype=torch.bfloat16)
    codes, scales = codes_of(x.reshape(-1, 100))
    w = layer.weight
    want = ((codes * scales[:, None]).to(dev) @ w.dequantize(torch.float64).t() + lin.bias.double()).view(3, 5, 37)
    with torch.no_grad():
        y = layer(x)
        assert torch.equal(layer(x.transpose(0, 1)), y.transpose(0, 1))
    # One rounding (2^-8), and fp32's of scales and sums (dequantize rounds its products, too: 2^-24 of up to |w| |x| 100 terms).
    torch.testing.assert_close(y.double(), want, rtol=2.0 ** -8 * 1.01, atol=1e-5)
    # A change of type leaves scales and codes alone, a copy and a state dict carry them.
    for other in (copy.deepcopy(layer), layer.half().bfloat16()):
        assert other.weight.scales.dtype == torch.float32
        with torch.no_grad():
            assert torch.equal(other(x), y)
    fresh = Int8Linear(Int8Rows.from_codes(torch.zeros(37, 100, dtype=torch.int8, device=dev), torch.ones(37, device=dev)), lin.bias)
    fresh.load_state_dict(layer.state_dict())
    with torch.no_grad():
        assert torch.equal(fresh(x), y)
    back = layer.cpu()
    assert back.weight.device.type == "cpu"
    with torch.no_grad(), pytest.raises(RuntimeError):
        back(x.cpu())


def test_what_is_replaced(dev):
    model = nn.ModuleDict(dict(a=nn.Linear(32, 16, dtype=torch.bfloat16, device=dev), lm_head=nn.Linear(16, 8, dtype=torch.bfloat16, device=dev),
                               b=nn.Linear(16, 4, device=dev), c=LinearWithLoRA(nn.Linear(8, 8, dtype=torch.float16, device=dev))))
    assert quantize_base(model) == 2
    assert isinstance(model["a"], Int8Linear) and isinstance(model["c"].base_layer, Int8Linear)
    assert type(model["lm_head"]) is nn.Linear and type(model["b"]) is nn.Linear  # float32 stays
    assert quantize_base(model, skip=()) == 1


def test_inputs_of_any_layout(dev):
    """What nn.Linear takes: expanded rows, transposed ones, an empty batch."""
    g = torch.Generator("cpu").manual_seed(5)
    layer = Int8Linear.from_linear(nn.Linear(40, 17, device=dev, dtype=torch.bfloat16))
    x = torch.randn(6, 40, generator=g).bfloat16().to(dev)
    with torch.no_grad():
        y = layer(x)
        assert torch.equal(layer(x[:1].expand(5, 40)), y[:1].expand(5, 17))
        assert torch.equal(layer(x[0].expand(2, 3, 40)), y[0].expand(2, 3, 17))
        assert torch.equal(layer(x.t().contiguous().t()), y)
        assert torch.equal(layer(x[0]), y[0])
        assert layer(x[:0]).shape == (0, 17) and layer(x.view(2, 3, 40)[:, :0]).shape == (2, 0, 17)
