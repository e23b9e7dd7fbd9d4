"""Plain 64-bit forms of the paged KV cache's operators, and inputs for their tests."""

import math
import random

import torch


class Pages:
    """The page allocator, page by page."""

    def __init__(self, n, width, num_pages, page):
        self.page, self.width = page, width
        self.table = [[-1] * width for _ in range(n)]
        self.held = [0] * n
        self.stack = list(range(num_pages - 1, -1, -1))

    def step(self, start, new, rows):
        """(row_indptr, kv_lens, positions, slots, missing) of one call."""
        need = [min(-(-(s + c) // self.page), self.width) for s, c in zip(start, new)]
        freed = [self.table[i][j] for i in range(len(need)) for j in range(need[i], self.held[i])]
        given, missing = 0, 0
        for i, k in enumerate(need):
            if k <= self.held[i]:
                self.held[i] = k
                continue
            for j in range(self.held[i], k):
                if given < len(freed):
                    self.table[i][j] = freed[given]
                elif self.stack:
                    self.table[i][j] = self.stack.pop()
                else:
                    self.table[i][j] = -1
                    missing += 1
                    continue
                given += 1
                self.held[i] = j + 1
        self.stack += reversed(freed[given:])
        indptr, pos, slots = [0], [], []
        for i, (s, c) in enumerate(zip(start, new)):
            indptr.append(indptr[-1] + c)
            for p in range(s, s + c):
                j = p // self.page
                pg = self.table[i][j] if j < self.width and j < need[i] else -1
                pos.append(p)
                slots.append(pg * self.page + p % self.page if pg >= 0 else -1)
        pad = rows - len(pos)
        return indptr, [s + c for s, c in zip(start, new)], pos + [0] * pad, slots + [-1] * pad, missing


def attention(q, keys, values, table, start, new, scale):
    """Outputs [rows, heads * d] in float64, and sum_l w_l |v_l| beside them (what a rounding of the weights moves)."""
    pages, g, page, d = keys.shape
    h = q.shape[1] // d
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    row = 0
    for i, (s, c) in enumerate(zip(start, new)):
        if c == 0:
            continue
        at = torch.arange(s + c, device=q.device)
        pg, off = table[i].to(q.device).long()[at // page], at % page
        k = keys[pg, :, off].double()             # [L, g, d]
        v = values[pg, :, :, off].double()
        x = q[row:row + c].double().view(c, g, h // g, d)
        see = at[None] <= s + torch.arange(c, device=q.device)[:, None]
        for z in range(g):
            sc = (x[:, z].reshape(-1, d) @ k[:, z].t().contiguous()).view(c, h // g, -1) * scale
            w = torch.softmax(sc.masked_fill(~see[:, None], -math.inf), -1).view(-1, s + c)
            # positions that no row of the chunk sees hold anything; 0 * NaN must not reach a row
            vz = v[:, z]
            o = torch.zeros(w.shape[0], d, dtype=torch.float64, device=q.device)
            a = torch.zeros_like(o)
            clean = torch.where(torch.isfinite(vz), vz, 0.0)
            o += w @ clean
            a += w @ clean.abs()
            for l in torch.nonzero(~torch.isfinite(vz).all(1)).flatten().tolist():
                sees = see[:, l].repeat_interleave(h // g)
                bad = torch.where(torch.isfinite(vz[l]), 0.0, vz[l])
                o += torch.where(sees[:, None] & (bad != 0), w[:, l:l + 1] * bad, 0.0)
            sl = (slice(row, row + c), slice(z * (h // g) * d, (z + 1) * (h // g) * d))
            out[sl] = o.view(c, -1)
            spread[sl] = a.view(c, -1)
        row += c
    return out, spread


def bound(want, spread, dtype, longest, scale_of_scores=40.0):
    """What the kernel may be off by.  Weights are rounded to the data type for the product with V (half a step each:
    eps/2 * sum w |v|), the result once more.  A score's fp32 error moves its weight by 2^-24 times a few times its size
    (a dot product of up to 128 terms, scaled: 16 roundings in a tree of partial sums taken as a bound).  float16
    weights below 2^-14 are off by up to 2^-25 absolutely, of a sum of at least 1."""
    half = torch.finfo(dtype).eps / 2
    err = half * (spread * (1 + half) + want.abs()) + 16 * scale_of_scores * 2.0 ** -24 * spread
    if dtype == torch.float16:
        err = err + longest * 2.0 ** -25 * 4.0  # |v| up to about 4
    return err + 1e-30


def draw_table(n_pages_of, num_pages, seed):
    ids = list(range(num_pages))
    random.Random(seed).shuffle(ids)
    width = max(1, max(n_pages_of))
    table, at = [], 0
    for k in n_pages_of:
        table.append(ids[at:at + k] + [-1] * (width - k))
        at += k
    return torch.tensor(table, dtype=torch.int32), ids[at:]


def verify(target, draft, tokens, indptr, accept, last):
    """(accepted, tokens) by the definition, one draft and one column at a time in float64."""
    n, most = tokens.shape
    counts, rows = [], []
    for i in range(n):
        a, b = indptr[i], indptr[i + 1]
        if b <= a:
            counts.append(0)
            rows.append([-1] * (most + 1))
            continue
        k, took = min(b - a - 1, most), 0
        while took < k:
            x = int(tokens[i, took])
            if not 0 <= x < target.shape[1]:
                break
            q = float(draft[i, took, x]) if draft is not None else 1.0
            if not float(accept[i, took]) * q < float(target[a + took, x]):
                break
            took += 1
        p = target[a + took].double().cpu()
        p = torch.where(p > 0, p, 0.0)
        m = p
        if took < k:
            if draft is not None:
                r = target[a + took].double().cpu() - draft[i, took].double().cpu()
                r = torch.where(r > 0, r, 0.0)
            else:
                r = p.clone()
                if 0 <= int(tokens[i, took]) < r.numel():
                    r[int(tokens[i, took])] = 0.0
            if float(r.sum()) > 0:
                m = r
        cum = m.cumsum(0)
        live = torch.nonzero(m > 0).flatten()
        hit = torch.nonzero((cum > float(last[i]) * float(cum[-1])) & (m > 0)).flatten()
        x = int(hit[0]) if hit.numel() else int(live[-1]) if live.numel() else -1
        counts.append(took)
        rows.append(tokens[i, :took].tolist() + [x] + [-1] * (most - took))
    return counts, rows
