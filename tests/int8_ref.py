"""Quantised rows and their products in 64 bits, from the definitions."""

import torch

LEAST = 2.0 ** -100


def codes_of(x: torch.Tensor):
    """(codes, scales) of rows in float64; a row with an infinity or NaN has a NaN scale and codes that mean nothing (0)."""
    x = x.double().cpu()
    bad = ~torch.isfinite(x).all(1)
    x = torch.where(bad[:, None], 0.0, x)
    top = x.abs().amax(1, keepdim=True).clamp(min=LEAST)
    codes = torch.round(x * 127 / top)  # ties to even; x * 127 is exact
    return codes, torch.where(bad, torch.nan, top[:, 0] / 127)


def product(codes, scales, wcodes, wscales, bias=None):
    """(result, bound of the fp32 part's error).  The sum is exact; its conversion, two products and the two scales' own
    roundings are at most half a step of fp32 each, and so is the bias's sum."""
    y = codes @ wcodes.double().t() * scales[:, None] * wscales.double()[None]
    slack = 5.01 * 2.0 ** -24 * y.abs()
    if bias is not None:
        y = y + bias.double().cpu()
        slack = slack + 1.01 * 2.0 ** -24 * y.abs()
    return y, slack


def check(got: torch.Tensor, want: torch.Tensor, slack: torch.Tensor) -> None:
    """``got`` is ``want`` but for ``slack`` and one rounding to its type: half a step, of fp16 no less than half its least."""
    half = torch.finfo(got.dtype).eps / 2
    least = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -134
    got = got.detach().double().cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    room = slack + half * (want.abs() + slack) + least
    off = torch.where(nan, 0.0, (got - want).abs() - room)
    assert bool((off <= 0).all()), f"off by up to {float(off.max()):.3g} more than {float(room[~nan].max()):.3g}"
