"""Serving in 8 bits (the base model's products and the paged KV cache), for timing and for comparing outputs.

A case is a dict of plain values; ``kind`` names the operator that one pass calls:

* ``linear``  ``int8_linear``: rows of 16-bit activations, quantised to 8-bit integers with a scale each, times an 8-bit
              weight with a scale for each output channel.
* ``write``   ``rotary_paged_write_fp8``: rotary on a step's q and k, and k and v into their slots of a cache of e4m3
              codes with an exponent for each block of 16 positions of a key head.
* ``attend``  ``paged_attention_fp8``: every new token over its request's pages of such a cache, causally.

Lengths are texts such as ``"512*2,1*64"``: ``new`` the new tokens of each request in this step, ``cached`` the tokens
that it has in the cache before.  ``page`` is the positions of a page.  Pages lie in the pool in random order and the
pool has pages that no request holds.  With ``own`` false every operator is computed by elementary torch operations.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
THETA = 500000.0
BLOCK = 16                                              # positions that share an exponent
EXPONENTS = {"bf16": (-117, 120), "fp16": (-15, 8)}     # of a block's scale: what the data type holds exactly
LARGEST = {"bf16": math.inf, "fp16": 65520.0}           # what rounds to infinity in the data type
LEAST = 2.0 ** -100                                     # a row's least maximum


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # One request decoding: a projection of one token, the smallest call.
        dict(name="linear one token", kind="linear", rows=1, inner=4096, out=4096, bias=False, dtype="bf16"),
        # A decode batch through the fused gate and up projections.
        dict(name="linear decode", kind="linear", rows=64, inner=4096, out=28672, bias=False, dtype="bf16"),
        # Two prompts beside 64 decoding requests through the down projection.
        dict(name="linear mixed", kind="linear", rows=1088, inner=14336, out=4096, bias=False, dtype="bf16"),
        # The rows of a batch of prompts through the fused q, k and v projections: the largest product.
        dict(name="linear prompts", kind="linear", rows=4075, inner=4096, out=6144, bias=False, dtype="bf16"),
        # Odd sizes, with a bias, in fp16.
        dict(name="linear odd", kind="linear", rows=333, inner=1111, out=777, bias=True, dtype="fp16"),
        # The new tokens of 64 decoding requests into the cache: most blocks hold earlier tokens.
        dict(name="write decode", kind="write", cached="500*40,1311*24", new="1*64", page=16, heads=32, kv_heads=8, dim=128,
             dtype="bf16"),
        # The rows of a batch of prompts of very different lengths, three of them behind cached tokens.
        dict(name="write prompts", kind="write", cached="0*5,96,512,17", new="837,64,1024,391,702,133,498,426", page=32,
             heads=32, kv_heads=8, dim=128, dtype="bf16"),
        # One request decoding with a small model: all latency.
        dict(name="attend one token", kind="attend", cached="202", new="1", page=16, heads=4, kv_heads=2, dim=64,
             dtype="fp16"),
        # A decode batch of ragged lengths, the attention of one layer.
        dict(name="attend decode", kind="attend", cached="200*20,1311*16,520*12,2047*12,3985*4", new="1*64", page=16,
             heads=32, kv_heads=8, dim=128, dtype="bf16"),
        # Few requests with long contexts: one long axis and few rows.
        dict(name="attend long context", kind="attend", cached="32000,20011,8191", new="1*3", page=64, heads=32, kv_heads=8,
             dim=128, dtype="bf16"),
        # Continuous batching: two prompts beside 64 decoding requests.
        dict(name="attend mixed", kind="attend", cached="0*2,300*30,911*34", new="512*2,1*64", page=16, heads=32, kv_heads=8,
             dim=128, dtype="bf16"),
        # A long prompt's second chunk beside two smaller ones: the largest call.
        dict(name="attend chunk", kind="attend", cached="4096,1000,0", new="4096,777,1301", page=32, heads=32, kv_heads=8,
             dim=128, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(values):
    return ",".join(str(v) for v in values)


def draw(rng):
    limits = {}
    for c in listed():
        w, kind = work(c), c["kind"]
        b, f = limits.get(kind, (0, 0))
        limits[kind] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= limits[case["kind"]][0] and w["flops"] <= limits[case["kind"]][1]:
            return case


def _draw(rng):
    kind = rng.choice(("linear", "linear", "write", "attend", "attend"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "linear":
        inner = rng.choice((4096, 14336, 1024, 256, _log(rng, 16, 14336), _log(rng, 16, 14336)))
        out = rng.choice((4096, 6144, 28672, 1024, _log(rng, 1, 28672), _log(rng, 1, 28672)))
        return dict(kind=kind, rows=_log(rng, 1, 6144), inner=inner, out=out, bias=rng.random() < 0.3, dtype=dtype)
    heads, kv_heads, dim = rng.choice(((32, 8, 128), (32, 8, 128), (16, 4, 128), (4, 2, 64), (8, 8, 64), (8, 1, 128),
                                       (12, 2, 64), (28, 4, 128), (32, 2, 64), (5, 1, 128)))
    page = rng.choice((16, 16, 32, 64, 128))
    step = rng.choice(("decode", "decode", "drafts", "prompts", "mixed", "mixed"))
    n = _log(rng, 1, 16 if step == "prompts" else 160)
    longest = _log(rng, 32, 8192)
    new, cached = [], []
    for i in range(n):
        prompt = step == "prompts" or (step == "mixed" and (i == 0 or rng.random() < 0.1))
        new.append(_log(rng, 1, 2048) if prompt else rng.randint(1, 9) if step == "drafts" else 1)
        cached.append(0 if prompt and rng.random() < 0.6 else _log(rng, 1, longest))
        if rng.random() < 0.05:
            new[-1] = 0  # a request that waits
    if not any(new):
        new[0] = 1
    return dict(kind=kind, cached=_text(cached), new=_text(new), page=page, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype)


def work(case):
    """The bytes and operations of one pass that the operator cannot do without."""
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["inner"], case["out"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    new, cached = _lens(case["new"]), _lens(case["cached"])
    rows = sum(new)
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "write":
        # The rows and their tables in, q and the codes out; a block's exponents are small beside them.
        return {"bytes": 2 * rows * (h + 2 * g) * d + 2 * 2 * rows * d + 4 * rows + 2 * rows * h * d + 2 * rows * g * d,
                "flops": 6 * rows * (h + g) * d}
    kv = sum(c + t for c, t in zip(cached, new) if t)
    pairs = sum(t * c + t * (t + 1) // 2 for c, t in zip(cached, new))
    return {"bytes": 2 * 2 * rows * h * d + 2 * kv * g * d + 2 * -(-kv // BLOCK) * g + 4 * -(-kv // case["page"]),
            "flops": 4 * h * d * pairs}


# ---------------------------------------------------------------- inputs
def _lens(text):
    out = []
    for part in str(text).split(","):
        v, _, times = part.partition("*")
        out += [int(v)] * int(times or 1)
    return out


def _gen(seed):
    return torch.Generator("cuda").manual_seed(int(seed))


def _randn(g, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _exponent(top, dtype):
    """The smallest e with top <= 448 * 2^e, within the data type's range."""
    m, x = torch.frexp(top)                   # top = m * 2^x, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = x - 9 + (m > 0.875).to(x.dtype)
    lo, hi = EXPONENTS[dtype]
    return torch.where(top > 0, e, lo).clamp(lo, hi)


def _e4m3(x, e, dtype):
    """x / 2^e rounded to the nearest number of 4 exponent and 3 mantissa bits, ties to even (as float8 values);
    infinities and NaN become NaN."""
    y = torch.ldexp(x, -e)
    _, p = torch.frexp(y)
    unit = (p - 1).clamp(min=-6) - 3          # exponent of the last bit's value
    y = torch.ldexp(torch.round(torch.ldexp(y, -unit)), unit)
    y = torch.where(e == EXPONENTS[dtype][1], y.clamp(-240, 240), y)  # 256 * 2^e is infinite in the data type
    return torch.where(x.abs() < LARGEST[dtype], y, torch.nan).float().to(torch.float8_e4m3fn)


def _quantised_rows(w):
    top = w.double().abs().amax(1, keepdim=True).clamp(min=LEAST)
    return torch.round(w.double() * 127 / top).to(torch.int8), (top[:, 0] / 127).float()


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "linear":
        m, k, n, dt = case["rows"], case["inner"], case["out"], DTYPES[case["dtype"]]
        # Activations behind a norm: one channel in a hundred is far larger than the others.
        gain = torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 8.0, 1.0)
        x = (_randn(g, (m, k), torch.float32) * gain).to(dt)
        codes, scales = _quantised_rows(_randn(g, (n, k), torch.float32, k ** -0.5))
        s = dict(case=case, x=x, bias=_randn(g, (n,), dt) if case["bias"] else None)
        if own:
            from multi_lora_amd.kernels import Int8Rows

            s["weight"] = Int8Rows.from_codes(codes, scales)
        else:
            s["codes"], s["scales"] = codes, scales
        return s
    new, cached, name = _lens(case["new"]), _lens(case["cached"]), case["dtype"]
    dt, h, kv, d, page = DTYPES[name], case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows = sum(new)
    lens = [c + t for c, t in zip(cached, new)]
    pool = sum(-(-t // page) for t in lens) + 8
    ids = list(range(pool))
    random.Random(seed).shuffle(ids)
    width = max(-(-t // page) for t in lens)
    table, at = [], 0
    for t in lens:
        held = -(-t // page)
        table.append(ids[at:at + held] + [-1] * (width - held))
        at += held
    # A cache that holds what blocks of rows were quantised to.
    blocks = page // BLOCK
    keys = _randn(g, (pool, kv, blocks, BLOCK, d), torch.float32)
    values = _randn(g, (pool, kv, d, blocks, BLOCK), torch.float32)
    ke = _exponent(keys.abs().amax((3, 4)), name)
    ve = _exponent(values.abs().amax((2, 4)), name)
    keys = _e4m3(keys, ke[..., None, None], name).view(pool, kv, page, d)
    values = _e4m3(values, ve[:, :, None, :, None], name).view(pool, kv, d, page)
    ke, ve = (ke + 127).to(torch.uint8), (ve + 127).to(torch.uint8)
    s = dict(case=case)
    if own:
        from multi_lora_amd.kernels import Fp8Pool, PageState, page_tables

        free = ids[at:]
        state = PageState(table=_i32(table), held=_i32([-(-t // page) for t in lens]),
                          free=_i32(free + [-1] * (pool - len(free))), counts=_i32([len(free), 0]), page=page)
        s["step"] = page_tables(state, _i32(cached), _i32(new), rows=rows, max_new=max(new), heads=h, kv_heads=kv, head_dim=d)
        s["pool"] = Fp8Pool(keys, values, ke, ve, dt)
    else:
        s.update(table=_i32(table), new=new, cached=cached, keys=keys, values=values, key_scales=ke, value_scales=ve)
        s["slots"] = torch.tensor([tab[(c + i) // page] * page + (c + i) % page for tab, c, t in zip(table, cached, new)
                                   for i in range(t)], device="cuda")
    if case["kind"] == "attend":
        s["q"] = _randn(g, (rows, h * d), dt, 1.5)
        return s
    qkv = _randn(g, (rows, (h + 2 * kv) * d), dt)  # the fused projection's output
    s["q"], s["k"], s["v"] = qkv.split((h * d, kv * d, kv * d), dim=1)
    pos = torch.tensor([c + i for c, t in zip(cached, new) for i in range(t)], dtype=torch.float64, device="cuda")
    ang = pos[:, None] * THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    s["cos"] = torch.cat((ang.cos(), ang.cos()), 1).to(dt)
    s["sin"] = torch.cat((-ang.sin(), ang.sin()), 1).to(dt)
    return s


# ---------------------------------------------------------------- the operators
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


def _own_linear(s):
    from multi_lora_amd.kernels import int8_linear

    return int8_linear(s["x"], s["weight"], s["bias"])


def _own_write(s):
    from multi_lora_amd.kernels import rotary_paged_write_fp8

    p = s["pool"]
    q = rotary_paged_write_fp8(s["q"], s["k"], s["v"], s["cos"], s["sin"], p, s["step"])
    return [q, p.keys, p.values, p.key_scales, p.value_scales]


def _own_attend(s):
    from multi_lora_amd.kernels import paged_attention_fp8

    return paged_attention_fp8(s["q"], s["pool"], s["step"], s["case"]["dim"] ** -0.5)


def _plain_linear(s):
    x = s["x"].float()
    top = x.abs().amax(1, keepdim=True).clamp(min=LEAST)
    codes = torch.round(x * 127 / top)  # x * 127 is exact in 32 bits for a 16-bit x: ties stay ties
    y = (codes @ s["codes"].float().t()) * (top / 127) * s["scales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _rotated(x, cos, sin, d):
    x = x.float().view(x.shape[0], -1, d)
    return x * cos.float()[:, None] + torch.cat((x[..., d // 2:], x[..., :d // 2]), -1) * sin.float()[:, None]


def _plain_write(s):
    case = s["case"]
    d, page, dt, slots, g, name = case["dim"], case["page"], DTYPES[case["dtype"]], s["slots"], case["kv_heads"], case["dtype"]
    rows = slots.shape[0]
    off = slots % BLOCK
    first = (off == 0) | (slots != torch.cat((slots.new_full((1,), -2), slots[:-1])) + 1)
    tile = first.cumsum(0) - 1                                          # the row's block among those of this call
    begin = off.new_full((rows,), BLOCK).scatter_reduce(0, tile, off, "amin")  # its first new row
    pg, sub = slots // page, slots % page // BLOCK
    old = (torch.arange(BLOCK, device=off.device) < begin[:, None])     # [tile, position]: earlier rows
    at = torch.zeros_like(slots).scatter_(0, tile, torch.arange(rows, device=off.device))  # a row of each tile
    tp, ts = pg[at], sub[at]

    def store(codes, scales, x, shape):
        """x [rows, g, d] into the blocks of codes, seen as [page, g, block, position, d] by ``shape``."""
        view = shape(codes)
        fresh = x.new_zeros((rows, g, BLOCK, d))
        fresh[tile, :, off] = x
        finite = torch.where(fresh.abs() < LARGEST[name], fresh.abs(), 0).amax((2, 3))
        e0 = scales[tp, :, ts].int() - 127
        e = torch.where((begin > 0)[:, None], torch.maximum(e0, _exponent(finite, name)), _exponent(finite, name))
        was = view[tp, :, ts].float()
        moved = _e4m3(torch.ldexp(was, e0[..., None, None]), e[..., None, None], name)
        new = torch.zeros_like(old).index_put_((tile, off), old.new_ones(()))[:, None, :, None]
        done = torch.where(new, _e4m3(fresh, e[..., None, None], name).float(),
                           torch.where(old[:, None, :, None], moved.float(), was)).to(codes.dtype)
        # Every row writes its whole block: rows of one block write the same.
        view.view(torch.uint8)[pg, :, sub] = done.view(torch.uint8)[tile]
        scales[pg, :, sub] = (e + 127).to(torch.uint8)[tile]

    pool, blocks = s["keys"].shape[0], page // BLOCK
    k, v = _rotated(s["k"], s["cos"], s["sin"], d), s["v"].float().view(rows, g, d)
    store(s["keys"], s["key_scales"], k, lambda t: t.view(pool, g, blocks, BLOCK, d))
    store(s["values"], s["value_scales"], v, lambda t: t.view(pool, g, d, blocks, BLOCK).permute(0, 1, 3, 4, 2))
    q = _rotated(s["q"], s["cos"], s["sin"], d).to(dt).view(rows, -1)
    return [q, s["keys"], s["values"], s["key_scales"], s["value_scales"]]


def _gathered(s, table, dtype=torch.float32):
    """Keys and values [n, g, positions, d] of the requests with these table rows."""
    ids = table.clamp(min=0).long()
    n, g, d, page = ids.shape[0], s["case"]["kv_heads"], s["case"]["dim"], s["case"]["page"]
    blocks = page // BLOCK
    ke, ve = (torch.ldexp(torch.ones((), dtype=dtype, device=ids.device), s[w][ids].int() - 127) for w in ("key_scales", "value_scales"))
    k = s["keys"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).to(dtype).view(n, -1, g, blocks, BLOCK, d) * ke[..., None, None]
    v = s["values"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).to(dtype).view(n, -1, g, d, blocks, BLOCK) * ve[:, :, :, None, :, None]
    return k.permute(0, 2, 1, 3, 4, 5).reshape(n, g, -1, d), v.permute(0, 2, 1, 4, 5, 3).reshape(n, g, -1, d)


def _plain_attend(s):
    case = s["case"]
    h, g, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    new, cached = s["new"], s["cached"]
    begin = [0]
    for t in new:
        begin.append(begin[-1] + t)
    out = torch.empty_like(s["q"])

    def together(which):
        t, n = max(new[i] for i in which), max(new[i] + cached[i] for i in which)
        k, v = _gathered(s, s["table"][which, :-(-n // page)])
        k, v = k[:, :, :n], v[:, :, :n]
        c, a, m = (torch.tensor([f[i] for i in which], device=out.device)[:, None] for f in (cached, begin, new))
        j = torch.arange(t, device=out.device)[None]
        row = (a + j).clamp(max=out.shape[0] - 1)
        q = s["q"][row].float().view(-1, t, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(len(which) * g, -1, d).contiguous()
        scores = torch.bmm(q, k.reshape(-1, n, d).transpose(1, 2).contiguous()).mul_(d ** -0.5).view(-1, g, h // g, t, n)
        later = torch.arange(n, device=out.device) > (c + j)[..., None]
        scores.masked_fill_(later[:, None, None], float("-inf"))
        e = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        o = torch.bmm(e.view(-1, h // g * t, n), v.reshape(-1, n, d).contiguous()).view(-1, g, h // g, t, d) / e.sum(-1, keepdim=True)
        o = o.permute(0, 3, 1, 2, 4).reshape(-1, h * d).to(out.dtype)
        use = (j < m).reshape(-1)
        # Rows that a shorter request does not have go where its last one's does not: nowhere (its own row again).
        keep = torch.where(use, torch.arange(use.numel(), device=out.device),
                           (torch.arange(len(which), device=out.device)[:, None] * t + m - 1).expand(-1, t).reshape(-1))
        out[(a + torch.minimum(j, m - 1)).reshape(-1)] = o[keep]

    # Requests of a few rows at once, padded; those of many (their scores are what takes the room) one by one.
    few = [i for i, t in enumerate(new) if 0 < t <= 16]
    if few:
        together(few)
    for i, t in enumerate(new):
        if t > 16:
            together([i])
    return out


# ---------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    global own
    was, own = own, False
    try:
        return globals()["_exact_" + case["kind"]](case, prepare(case, seed))
    finally:
        own = was


def _exact_linear(case, s):
    x = s["x"].double()
    limit = torch.maximum(x.abs().max(dim=1).values, torch.full_like(x[:, 0], LEAST))
    ratio = x * 127.0 / limit[:, None]
    low = ratio.floor()
    over = ratio - low
    code = low + ((over > 0.5) | ((over == 0.5) & (low.remainder(2) == 1))).double()
    y = torch.mm(code, s["codes"].double().t().contiguous())
    y *= (limit / 127.0)[:, None] * s["scales"].double()[None]
    return y + s["bias"].double() if s["bias"] is not None else y


#: Every non-negative value of 4 exponent and 3 mantissa bits: subnormals, then 2^e * (1 + m / 8), without the NaN.
E4M3 = [m / 8 * 2.0 ** -6 for m in range(8)] + [2.0 ** (e - 7) * (1 + m / 8) for e in range(1, 16) for m in range(8)][:-1]


def _exact_write(case, s):
    d, page, g = case["dim"], case["page"], case["kv_heads"]
    cos, sin, half = s["cos"].double(), s["sin"].double(), case["dim"] // 2
    lo, hi = EXPONENTS[case["dtype"]]

    def turn(x):
        x = x.double().view(x.shape[0], -1, d)
        y = torch.empty_like(x)
        y[..., :half] = x[..., :half] * cos[:, None, :half] + x[..., half:] * sin[:, None, :half]
        y[..., half:] = x[..., half:] * cos[:, None, half:] + x[..., :half] * sin[:, None, half:]
        return y

    table = torch.tensor(E4M3, dtype=torch.float64, device="cuda")

    def nearest(x):
        """The index of the nearest entry of the table, the even one of two; its sign apart."""
        a = x.abs().clamp(max=448.0).contiguous()
        up = torch.searchsorted(table, a).clamp(max=len(E4M3) - 1)
        down = (up - 1).clamp(min=0)
        du, dd = table[up] - a, a - table[down]
        index = torch.where((dd < du) | ((dd == du) & (down % 2 == 0)), down, up)
        return torch.copysign(table[index], x)

    slots = s["slots"].tolist()
    # The blocks of this call: (page, block), positions and rows.
    blocks = []
    for r, slot in enumerate(slots):
        if slot % BLOCK == 0 or r == 0 or slots[r - 1] + 1 != slot:
            blocks.append((slot // page, slot % page // BLOCK, []))
        blocks[-1][2].append((slot % BLOCK, r))
    new = {"k": turn(s["k"]), "v": s["v"].double().view(len(slots), g, d)}
    out = []
    for name, codes, scales in (("k", s["keys"].double(), s["key_scales"]), ("v", s["values"].double(), s["value_scales"])):
        codes = codes if name == "k" else codes.transpose(2, 3).contiguous()  # [pool, g, page, d]
        exps = scales.double() - 127
        tp, tb = (torch.tensor([b[i] for b in blocks], device="cuda") for i in (0, 1))
        begin = torch.tensor([b[2][0][0] for b in blocks], device="cuda")
        rows = torch.tensor([[dict(b[2]).get(i, -1) for i in range(BLOCK)] for b in blocks], device="cuda")
        here = rows >= 0
        x = new[name][rows.clamp(min=0)] * here[:, :, None, None]             # [block, position, g, d]
        place = tb[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")[None]
        was = codes[tp[:, None], :, place]                                    # [block, position, g, d]
        e0 = exps[tp, :, tb]                                                  # [block, g]
        top = x.abs().amax((1, 3))
        need = torch.ceil(torch.log2((top / 448.0).clamp(min=2.0 ** -1000)))
        need = need + (448.0 * torch.exp2(need) < top).double() - (448.0 * torch.exp2(need - 1) >= top).double()  # the logarithm's last bit
        need = torch.where(top > 0, need, torch.full_like(need, lo)).clamp(lo, hi)
        e = torch.where((begin > 0)[:, None], torch.maximum(e0, need), need)
        scale = torch.exp2(e)[:, None, :, None]
        y = nearest(x / scale)
        y = torch.where(e[:, None, :, None] == hi, y.clamp(-240, 240), y)
        moved = nearest(was * torch.exp2(e0)[:, None, :, None] / scale)
        before = (torch.arange(BLOCK, device="cuda")[None] < begin[:, None])[:, :, None, None]
        codes[tp[:, None], :, place] = torch.where(here[:, :, None, None], y, torch.where(before, moved, was))
        exps[tp, :, tb] = e
        out += [codes if name == "k" else codes.transpose(2, 3).contiguous(), (exps + 127).to(torch.uint8)]
    return [turn(s["q"]).reshape(len(slots), -1), out[0], out[2], out[1], out[3]]


def _exact_attend(case, s):
    h, g, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    keys, values = s["keys"].view(torch.uint8), s["values"].view(torch.uint8)
    row = 0
    for i, (t, c) in enumerate(zip(s["new"], s["cached"])):
        if t == 0:
            continue
        at = torch.arange(c + t, device="cuda")
        pg, off = s["table"][i, at // page].long(), at % page
        for u in range(g):
            ke = torch.exp2(s["key_scales"][pg, u, off // BLOCK].double() - 127)
            ve = torch.exp2(s["value_scales"][pg, u, off // BLOCK].double() - 127)
            k = keys[pg, u, off].view(torch.float8_e4m3fn).double() * ke[:, None]
            v = values[pg, u, :, off].contiguous().view(torch.float8_e4m3fn).double() * ve[:, None]
            for head in range(u * (h // g), (u + 1) * (h // g)):
                for r in range(0, t, 2048):
                    m = min(2048, t - r)
                    x = s["q"][row + r:row + r + m, head * d:(head + 1) * d].double() @ k.t() * d ** -0.5
                    x += torch.triu(torch.full_like(x, -math.inf), diagonal=c + r + 1)
                    out[row + r:row + r + m, head * d:(head + 1) * d] = torch.softmax(x, 1) @ v
        row += t
    return out
