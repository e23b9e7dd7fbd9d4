"""The paged KV cache's operators as a serving program calls them, for timing and for comparing outputs.

A case is a dict of plain values; ``kind`` names the operator that one pass calls:

* ``tables``  ``page_tables`` twice: pages, slots, positions and the attention's work list of a step's new tokens, then
              the step taken back (a rejected draft, a preempted request), which returns the pages.
* ``write``   ``rotary_paged_write``: rotary on a step's q and k, and k and v into their slots of the cache.
* ``attend``  ``paged_attention``: every new token over its request's pages, causally.
* ``verify``  ``verify_drafts``: accepted drafts and the token after them, from given random numbers.

Lengths are texts such as ``"512*2,1*64"``: ``new`` the new tokens of each request in this step, ``cached`` the tokens
that it has in the cache before.  ``page`` is the positions of a page.  Pages lie in the pool in random order and the
pool has pages that no request holds.  With ``own`` false every operator is computed by elementary torch operations.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
THETA = 500000.0


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # A decode step of a large batch: one token a request, a few of which begin a page.
        dict(name="tables decode", kind="tables", cached="200*40,333*21,1024*32,75*60,4095*3,16*12", new="1*168", page=16,
             heads=32, kv_heads=8, dim=128),
        # A step that admits prompts beside decoding requests: thousands of rows.
        dict(name="tables mixed", kind="tables", cached="0*6,96,512,700*64", new="837,64,1024,391,702,133,498,426,1*64",
             page=16, heads=32, kv_heads=8, dim=128),
        # The new tokens of 64 decoding requests into the cache.
        dict(name="write decode", kind="write", cached="500*40,1311*24", new="1*64", page=16, heads=32, kv_heads=8, dim=128,
             dtype="bf16"),
        # The rows of a batch of prompts of very different lengths.
        dict(name="write prompts", kind="write", cached="0*5,96,512,17", new="837,64,1024,391,702,133,498,426", page=16,
             heads=32, kv_heads=8, dim=128, dtype="bf16"),
        # One request decoding with a small model: the smallest call, all latency.
        dict(name="attend one token", kind="attend", cached="202", new="1", page=16, heads=4, kv_heads=2, dim=64,
             dtype="fp16"),
        # A decode batch of ragged lengths, the attention of one layer.
        dict(name="attend decode", kind="attend", cached="200*20,1311*16,520*12,2047*12,3985*4", new="1*64", page=16,
             heads=32, kv_heads=8, dim=128, dtype="bf16"),
        # Few requests with long contexts: one long axis and few rows.
        dict(name="attend long context", kind="attend", cached="32000,20011,8191", new="1*3", page=64, heads=32, kv_heads=8,
             dim=128, dtype="bf16"),
        # Verification of four drafted tokens a request.
        dict(name="attend drafts", kind="attend", cached="200*16,777*10,1500*6", new="5*32", page=16, heads=16, kv_heads=4,
             dim=128, dtype="fp16"),
        # Continuous batching: two prompts beside 64 decoding requests.
        dict(name="attend mixed", kind="attend", cached="0*2,300*30,911*34", new="512*2,1*64", page=16, heads=32, kv_heads=8,
             dim=128, dtype="bf16"),
        # A long prompt's second chunk beside two smaller ones: the largest call.
        dict(name="attend chunk", kind="attend", cached="4096,1000,0", new="4096,777,1301", page=32, heads=32, kv_heads=8,
             dim=128, dtype="bf16"),
        # Four drafted tokens of one request over a small vocabulary.
        dict(name="verify one", kind="verify", drafts="4", vocab=4096, dtype="fp32", draft_probs=True),
        # Drafts of 32 requests over a large vocabulary; some requests have none.
        dict(name="verify batch", kind="verify", drafts="4*26,2*4,0*2", vocab=128256, dtype="fp32", draft_probs=True),
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
    kind = rng.choice(("tables", "write", "attend", "attend", "attend", "verify"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "verify":
        n = _log(rng, 1, 64)
        return dict(kind=kind, drafts=_text(rng.randint(0, 8) for _ in range(n)), vocab=_log(rng, 512, 128256),
                    dtype=rng.choice(("fp32", "fp32", "bf16", "fp16")), draft_probs=rng.random() < 0.7)
    heads, kv_heads, dim = rng.choice(((32, 8, 128), (32, 8, 128), (16, 4, 128), (4, 2, 64), (8, 8, 64), (8, 1, 128),
                                       (12, 2, 64), (28, 4, 128), (32, 2, 64), (5, 1, 128)))
    page = rng.choice((8, 16, 16, 32, 64, 128))
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
    case = dict(kind=kind, cached=_text(cached), new=_text(new), page=page, heads=heads, kv_heads=kv_heads, dim=dim)
    if kind != "tables":
        case["dtype"] = dtype
    return case


def work(case):
    """The bytes and operations of one pass that the operator cannot do without."""
    if case["kind"] == "verify":
        # One row of the target's probabilities a request and, where it has drafts, one of the draft's (a request whose
        # drafts are all accepted needs none, which only the random numbers know).
        drafts = _lens(case["drafts"])
        rows = len(drafts) + (sum(k > 0 for k in drafts) if case["draft_probs"] else 0)
        return {"bytes": rows * case["vocab"] * SIZES[case["dtype"]], "flops": 2 * rows * case["vocab"]}
    new, cached = _lens(case["new"]), _lens(case["cached"])
    rows, n, page = sum(new), len(new), case["page"]
    h, g, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "tables":
        taken = sum(-(-(c + t) // page) - -(-c // page) for c, t in zip(cached, new))
        return {"bytes": 4 * (2 * rows + 6 * n + 4 * taken), "flops": 0}
    size = SIZES[case["dtype"]]
    if case["kind"] == "write":
        return {"bytes": 2 * rows * (h + 2 * g) * d * size + 2 * rows * d * size + 4 * rows, "flops": 6 * rows * (h + g) * d}
    kv = sum(c + t for c, t in zip(cached, new) if t)
    pairs = sum(t * c + t * (t + 1) // 2 for c, t in zip(cached, new))
    return {"bytes": 2 * rows * h * d * size + 2 * kv * g * d * size + 4 * -(-kv // page), "flops": 4 * h * d * pairs}


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


def _pages(case, seed, tokens):
    """Page ids of each request for ``tokens[i]`` positions, and the free ones, in random order."""
    need = [-(-t // case["page"]) for t in tokens]
    lens = [c + t for c, t in zip(_lens(case["cached"]), _lens(case["new"]))]
    pool = sum(-(-t // case["page"]) for t in lens) + 8
    ids = list(range(pool))
    random.Random(seed).shuffle(ids)
    width = max(-(-t // case["page"]) for t in lens)
    table, at = [], 0
    for k in need:
        table.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    return table, need, ids[at:], pool


def _cache_state(case, seed, tokens):
    """The allocator's state in which every request holds the pages of ``tokens[i]`` positions."""
    table, held, free, pool = _pages(case, seed, tokens)
    s = dict(table=_i32(table), held=_i32(held), free=_i32(free + [-1] * (pool - len(free))), counts=_i32([len(free), 0]),
             page=case["page"])
    if own:
        from multi_lora_amd.kernels import PageState

        s = PageState(**s)
    return s, pool


def _tables_args(case):
    new, cached = _lens(case["new"]), _lens(case["cached"])
    return dict(start=_i32(cached), new=_i32(new), rows=sum(new), max_new=max(new), heads=case["heads"],
                kv_heads=case["kv_heads"], head_dim=case["dim"])


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "verify":
        return _prepare_verify(case, g)
    new, cached = _lens(case["new"]), _lens(case["cached"])
    if case["kind"] == "tables":
        state, _ = _cache_state(case, seed, cached)
        return dict(case=case, state=state, args=_tables_args(case))
    dt, h, kv, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    rows = sum(new)
    state, pool = _cache_state(case, seed, [c + t for c, t in zip(cached, new)])
    s = dict(case=case, keys=_randn(g, (pool, kv, case["page"], d), dt), values=_randn(g, (pool, kv, d, case["page"]), dt))
    if own:
        from multi_lora_amd.kernels import page_tables

        a = _tables_args(case)
        s["batch"] = page_tables(state, a.pop("start"), a.pop("new"), **a)
    else:
        s["table"] = state["table"]
        s["new"], s["cached"] = new, cached
    if case["kind"] == "attend":
        s["q"] = _randn(g, (rows, h * d), dt, 1.5)
        return s
    qkv = _randn(g, (rows, (h + 2 * kv) * d), dt)  # the fused projection's output
    s["q"], s["k"], s["v"] = qkv.split((h * d, kv * d, kv * d), dim=1)
    pos = torch.tensor([c + i for c, t in zip(cached, new) for i in range(t)], dtype=torch.float64, device="cuda")
    ang = pos[:, None] * THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    s["cos"] = torch.cat((ang.cos(), ang.cos()), 1).to(dt)
    s["sin"] = torch.cat((-ang.sin(), ang.sin()), 1).to(dt)
    s["slots"] = s["batch"].slots if own else _i32([tab[(c + i) // case["page"]] * case["page"] + (c + i) % case["page"]
                                                    for tab, c, t in zip(_pages(case, seed, [c + t for c, t in zip(cached, new)])[0],
                                                                         cached, new) for i in range(t)])
    return s


def _prepare_verify(case, g):
    drafts, v, dt = _lens(case["drafts"]), case["vocab"], DTYPES[case["dtype"]]
    n, most, rows = len(drafts), max(1, max(drafts)), sum(drafts) + len(drafts)
    logits = _randn(g, (rows, v), torch.float32, 3.0)
    indptr = [0]
    for k in drafts:
        indptr.append(indptr[-1] + k + 1)
    # Draft row j of request i proposes from logits near the target's row j (the last one repeats where it has fewer).
    at = torch.tensor([[min(indptr[i] + j, indptr[i + 1] - 1) for j in range(most)] for i in range(n)], device="cuda")
    near = logits[at] + _randn(g, (n, most, v), torch.float32, 0.5)
    q = torch.softmax(near, -1).to(dt)
    noise = torch.empty((n, most, v), device="cuda").exponential_(generator=g)
    tokens = (q.float() / noise).argmax(-1)  # drawn from q
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    return dict(case=case, target=torch.softmax(logits, -1).to(dt), draft=q if case["draft_probs"] else None, tokens=tokens,
                indptr=_i32(indptr), accept=rand(n, most), last=rand(n))


# ---------------------------------------------------------------- the operators
def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


def _own_tables(s):
    from multi_lora_amd.kernels import page_tables

    a = dict(s["args"])
    start, new = a.pop("start"), a.pop("new")
    b = page_tables(s["state"], start, new, **a)
    page_tables(s["state"], start, torch.zeros_like(new), rows=0, max_new=0)
    st = s["state"]
    return [b.row_indptr, b.kv_lens, b.positions, b.slots, st.table, st.held, st.free[:_live(s)], st.counts]


def _own_write(s):
    from multi_lora_amd.kernels import rotary_paged_write

    q = rotary_paged_write(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["keys"], s["values"], s["slots"])
    return [q, s["keys"], s["values"]]


def _own_attend(s):
    from multi_lora_amd.kernels import paged_attention

    return paged_attention(s["q"], s["keys"], s["values"], s["batch"], s["case"]["dim"] ** -0.5)


def _own_verify(s):
    from multi_lora_amd.kernels import verify_drafts

    return list(verify_drafts(s["target"], s["draft"], s["tokens"], s["indptr"], s["accept"], s["last"]))


def _live(s):
    """Free pages once the step is taken back: what the stack holds below its top."""
    case = s["case"]
    lens = [c + t for c, t in zip(_lens(case["cached"]), _lens(case["new"]))]
    return 8 + sum(-(-t // case["page"]) - -(-c // case["page"]) for t, c in zip(lens, _lens(case["cached"])))


def _step_tables(st, start, new):
    """One call of the page tables: ``st`` is changed in place; returns what describes the new rows."""
    table, held, free, counts, page = st["table"], st["held"], st["free"], st["counts"], st["page"]
    width, pool = table.shape[1], free.shape[0]
    total = start + new
    need = ((total + page - 1) // page).clamp(max=width)
    freed, taken = (held - need).clamp(min=0).long(), (need - held).clamp(min=0).long()
    freed0, taken0 = freed.cumsum(0) - freed, taken.cumsum(0) - taken
    top, nf, nt = counts[0].long(), freed.sum(), taken.sum()
    j = torch.arange(width, device=table.device)[None]
    # Freed pages, listed in order; taken page a is freed page a, or the stack's entry below its top.
    goes = (j >= need[:, None]) & (j < held[:, None])
    at = torch.where(goes, freed0[:, None] + j - need[:, None], pool)
    listed_ = torch.full((pool + 1,), -1, dtype=table.dtype, device=table.device)
    listed_.scatter_(0, at.reshape(-1).clamp(max=pool), torch.where(goes, table, -1).reshape(-1))
    comes = (j >= held[:, None]) & (j < need[:, None])
    a = torch.where(comes, taken0[:, None] + j - held[:, None], 0)
    below = top - 1 - (a - nf)
    page_of = torch.where(a < nf, listed_[a.clamp(max=pool)], torch.where(below >= 0, free[below.clamp(0, pool - 1)], -1))
    table.copy_(torch.where(comes, page_of, table))
    # What nobody took goes on the stack, the last one first.
    f = torch.arange(pool, device=table.device)
    stay = (f >= nt) & (f < nf)
    to = torch.where(stay, top + nf - 1 - f, pool)
    room = torch.cat((free, free.new_full((1,), -1)))
    room.scatter_(0, to, torch.where(stay, listed_[:pool], -1))
    free.copy_(room[:pool])
    got = torch.minimum(taken, (top + nf - taken0).clamp(min=0))
    held.copy_(torch.where(need > held, held + got, need))
    counts.copy_(torch.stack(((top + nf - nt).clamp(min=0), (nt - top - nf).clamp(min=0))))
    return total


def _plain_tables(s):
    st, a = s["state"], s["args"]
    start, new, rows, page = a["start"], a["new"], a["rows"], st["page"]
    total = _step_tables(st, start, new)
    ends = new.cumsum(0)
    indptr = torch.cat((ends.new_zeros(1), ends)).to(torch.int32)
    r = torch.arange(rows, device=ends.device)
    i = torch.searchsorted(ends, r, right=True)
    pos = start[i] + (r - indptr[i])
    slots = st["table"][i, (pos // page).long()] * page + pos % page
    _step_tables(st, start, torch.zeros_like(new))
    return [indptr, total, pos.to(torch.int32), slots.to(torch.int32), st["table"], st["held"], st["free"][:_live(s)],
            st["counts"]]


def _rotated(x, cos, sin, d):
    x = x.float().view(x.shape[0], -1, d)
    return x * cos.float()[:, None] + torch.cat((x[..., d // 2:], x[..., :d // 2]), -1) * sin.float()[:, None]


def _plain_write(s):
    case = s["case"]
    d, page, dt, rows = case["dim"], case["page"], DTYPES[case["dtype"]], s["q"].shape[0]
    pg, off = (s["slots"] // page).long(), (s["slots"] % page).long()
    s["keys"][pg, :, off] = _rotated(s["k"], s["cos"], s["sin"], d).to(dt)
    s["values"][pg, :, :, off] = s["v"].reshape(rows, -1, d)
    return [_rotated(s["q"], s["cos"], s["sin"], d).to(dt).view(rows, -1), s["keys"], s["values"]]


def _plain_attend(s):
    case = s["case"]
    h, g, d, dt = case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    out = torch.empty_like(s["q"])
    row = 0
    for i, (t, c) in enumerate(zip(s["new"], s["cached"])):
        if t == 0:
            continue
        n = c + t
        ids = s["table"][i, :-(-n // case["page"])].long()
        k = s["keys"][ids].float().permute(1, 3, 0, 2).reshape(g, d, -1)[:, :, :n].contiguous()
        v = s["values"][ids].float().permute(1, 0, 3, 2).reshape(g, -1, d)[:, :n].contiguous()
        q = s["q"][row:row + t].float().view(t, g, h // g, d).permute(1, 2, 0, 3).reshape(g, -1, d).contiguous()
        scores = torch.bmm(q, k).mul_(d ** -0.5).view(g, h // g, t, n)
        later = torch.arange(n, device=q.device)[None] > c + torch.arange(t, device=q.device)[:, None]
        scores.masked_fill_(later, float("-inf"))
        e = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        o = torch.bmm(e.view(g, -1, n), v).view(g, h // g, t, d) / e.sum(-1, keepdim=True)
        out[row:row + t] = o.permute(2, 0, 1, 3).reshape(t, h * d).to(dt)
        row += t
    return out


def _plain_verify(s):
    target, draft, tokens, indptr = s["target"], s["draft"], s["tokens"], s["indptr"].long()
    (n, most), v = tokens.shape, target.shape[1]
    first, k = indptr[:-1], indptr[1:] - indptr[:-1] - 1
    j = torch.arange(most, device=tokens.device)[None]
    p = target[(first[:, None] + j).clamp(max=target.shape[0] - 1), tokens].double()
    q = draft.gather(2, tokens[..., None])[..., 0].double() if draft is not None else torch.ones_like(p)
    ok = (s["accept"].double() * q < p) & (j < k[:, None])
    accepted = ok.long().cumprod(1).sum(1)
    rows = target[first + accepted].double()
    at = accepted.clamp(max=most - 1)
    i = torch.arange(n, device=tokens.device)
    less = draft[i, at].double() if draft is not None else torch.zeros_like(rows).scatter_(1, tokens[i, at][:, None], 1.0)
    rest = (rows - less).clamp(min=0)
    use = (accepted < k) & (rest.sum(1) > 0)
    cum = torch.where(use[:, None], rest, rows).cumsum(1)
    last = (cum <= s["last"].double()[:, None] * cum[:, -1:]).sum(1)
    out = torch.where(j < accepted[:, None], tokens, -1)
    out = torch.cat((out, out.new_full((n, 1), -1)), 1)
    out.scatter_(1, accepted[:, None], last[:, None])
    return [accepted.to(torch.int32), out]


# ---------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    global own
    was, own = own, False
    try:
        return globals()["_exact_" + case["kind"]](case, prepare(case, seed))
    finally:
        own = was


def _exact_tables(case, s):
    new, cached, page = _lens(case["new"]), _lens(case["cached"]), case["page"]
    table, stack = s["state"]["table"].tolist(), s["state"]["free"].tolist()[:int(s["state"]["counts"][0])]
    held, before = s["state"]["held"].tolist(), list(stack)
    indptr, pos, slots = [0], [], []
    for i, (c, t) in enumerate(zip(cached, new)):
        for j in range(held[i], -(-(c + t) // page)):
            table[i][j] = stack.pop()
        for at in range(c, c + t):
            pos.append(at)
            slots.append(table[i][at // page] * page + at % page)
        indptr.append(indptr[-1] + t)
    # Taken back: every page returns to where it was taken from.
    return [_i32(indptr), _i32([c + t for c, t in zip(cached, new)]), _i32(pos), _i32(slots), _i32(table), _i32(held),
            _i32(before), _i32([len(before), 0])]


def _exact_write(case, s):
    d, page = case["dim"], case["page"]
    cos, sin = s["cos"].double(), s["sin"].double()
    half = d // 2

    def turn(x):
        x = x.double().view(x.shape[0], -1, d)
        y = torch.empty_like(x)
        y[..., :half] = x[..., :half] * cos[:, None, :half] + x[..., half:] * sin[:, None, :half]
        y[..., half:] = x[..., half:] * cos[:, None, half:] + x[..., :half] * sin[:, None, half:]
        return y

    keys, values = s["keys"].double(), s["values"].double()
    slots = s["slots"].long()
    flat = keys.transpose(1, 2).reshape(-1, keys.shape[1], d)          # [pool * page, kv_heads, d]
    flat[slots] = turn(s["k"])
    keys = flat.view(-1, page, keys.shape[1], d).transpose(1, 2).contiguous()
    flat = values.permute(0, 3, 1, 2).reshape(-1, values.shape[1], d)
    flat[slots] = s["v"].double().reshape(slots.shape[0], -1, d)
    values = flat.view(-1, page, values.shape[1], d).permute(0, 2, 3, 1).contiguous()
    return [turn(s["q"]).reshape(slots.shape[0], -1), keys, values]


def _exact_attend(case, s):
    h, g, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for i, (t, c) in enumerate(zip(s["new"], s["cached"])):
        if t == 0:
            continue
        at = torch.arange(c + t, device="cuda")
        pg, off = s["table"][i, at // page].long(), at % page
        for head in range(h):
            k = s["keys"][pg, head // (h // g), off].double()
            v = s["values"][pg, head // (h // g), :, off].double()
            for r in range(0, t, 2048):
                m = min(2048, t - r)
                x = s["q"][row + r:row + r + m, head * d:(head + 1) * d].double() @ k.t() * d ** -0.5
                x += torch.triu(torch.full_like(x, -math.inf), diagonal=c + r + 1)
                out[row + r:row + r + m, head * d:(head + 1) * d] = torch.softmax(x, 1) @ v
        row += t
    return out


def _exact_verify(case, s):
    target, tokens, indptr = s["target"], s["tokens"].tolist(), s["indptr"].tolist()
    u, w = s["accept"].tolist(), s["last"].tolist()
    counts, rows = [], []
    for i, (a, b) in enumerate(zip(indptr, indptr[1:])):
        took = 0
        while took < b - a - 1:
            x = tokens[i][took]
            q = float(s["draft"][i, took, x]) if s["draft"] is not None else 1.0
            if not u[i][took] * q < float(target[a + took, x]):
                break
            took += 1
        mass = target[a + took].double()
        if took < b - a - 1:
            if s["draft"] is not None:
                less = torch.relu(mass - s["draft"][i, took].double())
            else:
                less = mass.clone()
                less[tokens[i][took]] = 0
            mass = less if float(less.sum()) > 0 else mass
        cum = torch.cumsum(mass, 0)
        x = int(torch.nonzero(cum > w[i] * float(cum[-1]))[0])
        counts.append(took)
        rows.append(tokens[i][:took] + [x] + [-1] * (len(tokens[i]) - took))
    return [_i32(counts), torch.tensor(rows, dtype=torch.int64, device="cuda")]
