"""The 8-bit cache's write from its definition, block by block in 64 bits."""

import math

import torch

BLOCK = 16
RANGE = {torch.bfloat16: (-117, 120), torch.float16: (-15, 8)}
END = {torch.bfloat16: math.inf, torch.float16: 65520.0}
# Every non-negative e4m3 number by its code: subnormals, then 2^e * (1 + m / 8), the last of them 448.
NUMBERS = [m / 8 * 2.0 ** -6 for m in range(8)] + [2.0 ** (e - 7) * (1 + m / 8) for e in range(1, 16) for m in range(8)][:-1]
TABLE = torch.tensor(NUMBERS, dtype=torch.float64)


def encode(y: torch.Tensor) -> torch.Tensor:
    """Codes (uint8) of the nearest numbers, ties to the even code; NaN is 0x7f."""
    nan = torch.isnan(y)
    a = torch.where(nan, 0.0, y).abs().clamp(max=448.0).contiguous()
    up = torch.searchsorted(TABLE, a).clamp(max=len(NUMBERS) - 1)
    down = (up - 1).clamp(min=0)
    du, dd = TABLE[up] - a, a - TABLE[down]
    c = torch.where((dd < du) | ((dd == du) & (down % 2 == 0)), down, up)
    c = torch.where(nan, 0x7f, c)
    return (c + torch.where(torch.signbit(y) & ~nan, 128, 0)).to(torch.uint8)


def decode(codes: torch.Tensor) -> torch.Tensor:
    c = codes.long()
    v = TABLE[(c & 127).clamp(max=len(NUMBERS) - 1)]
    v = torch.where((c & 127) == 127, torch.nan, v)
    return torch.where(c >= 128, -v, v)


def exponent(x: torch.Tensor, dtype) -> int:
    """The least e with max|x| <= 448 * 2^e over the numbers of x."""
    lo, hi = RANGE[dtype]
    a = x.abs()
    a = torch.where(a < END[dtype], a, 0.0)
    top = float(a.max())
    if top == 0:
        return lo
    e = math.frexp(top / 448.0)[1]
    while 448.0 * 2.0 ** (e - 1) >= top:
        e -= 1
    return min(max(e, lo), hi)


def quantise(x: torch.Tensor, e: int, dtype) -> torch.Tensor:
    y = x * 2.0 ** -e
    if e == RANGE[dtype][1]:
        y = y.clamp(-240.0, 240.0)
    return encode(torch.where(x.abs() < END[dtype], y, torch.nan))


def write(keys, values, key_scales, value_scales, k, v, slots, dtype):
    """The pools (uint8 codes and exponent bytes, on the CPU, changed in place) after a write of rotated ``k`` and ``v``
    ``[rows, kv_heads, d]`` (float64) into ``slots`` (a list, -1: none)."""
    page, kv_heads = keys.shape[2], keys.shape[1]
    end = keys.shape[0] * page
    r = 0
    while r < len(slots):
        if not 0 <= slots[r] < end:
            r += 1
            continue
        n = 1
        while r + n < len(slots) and slots[r + n] == slots[r] + n and (slots[r] + n) % BLOCK:
            n += 1
        pg, at = divmod(slots[r], page)
        off, b = at % BLOCK, at // BLOCK
        here, early = slice(at, at + n), slice(at - off, at)
        for g in range(kv_heads):
            for x, codes, scales in ((k[r:r + n, g], keys[pg, g], key_scales), (v[r:r + n, g], values[pg, g].t(), value_scales)):
                e, was = exponent(x, dtype), int(scales[pg, g, b]) - 127
                if off:
                    e = max(e, was)
                    if e > was:
                        codes[early] = encode(decode(codes[early]) * 2.0 ** (was - e))
                codes[here] = quantise(x, e, dtype)
                scales[pg, g, b] = e + 127
        r += n
