"""The paged KV cache in 8 bits, on the HIP kernels.

``rotary_paged_write_fp8`` and ``paged_attention_fp8`` are
``rotary_paged_write`` and ``paged_attention`` (``kernels/paged.py``) over an
``Fp8Pool``: e4m3 codes with an exponent for each block of 16 positions of a
key head, half the bytes of a 16-bit cache and of its attention.  Page tables
and steps are the same.

A code times its block's power of two is exactly a number of the cache's data
type, and attention multiplies with it; so what 8 bits cost is one rounding of
the rotated keys and of the values (a relative 2^-4 at most; 2^-10 of the
block's scale for the smallest numbers).  Blocks fill while requests decode:
an exponent grows with the largest row so far, and codes of earlier rows only
move theirs, so they keep their value unless it falls below the block's least
normal number, 2^-14 of its largest.

Float16 or bfloat16 data, ``d`` 64 or 128, pages of a power of two positions
from 16 to 1024.  There is no CPU path and no derivative in either mode:
inputs that ask for one are refused, and so are calls under a trace.

No counterpart in the reference, whose decode runs over
``transformers.StaticCache`` (multi_lora/graph_decode.py:23-111).
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import Optional, Tuple

import torch

from .. import _ffi
from .paged import (_DTYPES, PagedStep, _guard, _no_grad, _no_tangent, _on_gpu, _rows, _untraced, _writes)

BLOCK = 16   # positions that share an exponent
BIAS = 127   # a stored exponent byte is this much more


@dataclass(frozen=True)
class Fp8Pool:
    """One layer's pages: ``keys [num_pages, kv_heads, page, d]`` and ``values
    [num_pages, kv_heads, d, page]`` of e4m3 codes, ``key_scales`` and
    ``value_scales [num_pages, kv_heads, page / 16]`` of exponent bytes (uint8).
    A code ``c`` of a block with byte ``b`` stands for ``c * 2**(b - 127)``, a
    number of ``dtype``, the type of the rows that are written and attend."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scales: torch.Tensor
    value_scales: torch.Tensor
    dtype: torch.dtype
    _code: int = field(init=False, repr=False, compare=False)

    def __post_init__(self) -> None:
        k, v = self.keys, self.values
        if k.dim() != 4 or v.dim() != 4:
            raise ValueError("keys [num_pages, kv_heads, page, d] and values [num_pages, kv_heads, d, page]")
        pages, kv_heads, page, d = k.shape
        if tuple(v.shape) != (pages, kv_heads, d, page) or any(t.dtype != torch.float8_e4m3fn for t in (k, v)):
            raise ValueError(f"keys {tuple(k.shape)} {k.dtype}, values {tuple(v.shape)} {v.dtype}: float8_e4m3fn of one pool expected")
        if pages == 0 or kv_heads == 0 or not 16 <= page <= 1024 or page & (page - 1) or d not in (64, 128):
            raise ValueError(f"pages of a power of two positions from 16 to 1024 with heads of 64 or 128, got {tuple(k.shape)}")
        size = kv_heads * page * d
        for name, t in (("keys", k), ("values", v)):
            if not t[0].is_contiguous() or pages > 1 and (t.stride(0) < size or t.stride(0) % 16) or t.data_ptr() % 16:
                raise ValueError(f"{name}: every page must be contiguous, at a multiple of 16 bytes")
        for name, t in (("key_scales", self.key_scales), ("value_scales", self.value_scales)):
            if t.dtype != torch.uint8 or tuple(t.shape) != (pages, kv_heads, page // BLOCK) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 tensor of shape {(pages, kv_heads, page // BLOCK)}, got "
                                 f"{tuple(t.shape)} {t.dtype}")
        if any(t.device != k.device for t in (v, self.key_scales, self.value_scales)):
            raise ValueError("keys, values and scales must be on one device")
        if self.dtype not in _DTYPES:
            raise ValueError(f"float16 or bfloat16 rows, got {self.dtype}")
        object.__setattr__(self, "_code", _ffi.dtype_code(self.dtype))

    @classmethod
    def new(cls, num_pages: int, kv_heads: int, page: int, d: int, dtype: torch.dtype, device) -> "Fp8Pool":
        """A pool of zeros."""
        codes = dict(dtype=torch.uint8, device=device)
        return cls(torch.zeros((num_pages, kv_heads, page, d), **codes).view(torch.float8_e4m3fn),
                   torch.zeros((num_pages, kv_heads, d, page), **codes).view(torch.float8_e4m3fn),
                   torch.full((num_pages, kv_heads, page // BLOCK), BIAS, **codes),
                   torch.full((num_pages, kv_heads, page // BLOCK), BIAS, **codes), dtype)

    @property
    def shape(self) -> Tuple[int, int, int, int]:
        """``(num_pages, kv_heads, page, d)``."""
        return tuple(self.keys.shape)

    def dequantize(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The values that the codes stand for, as 16-bit pools of the same layout."""
        pages, g, page, d = self.keys.shape
        ke, ve = (s.to(torch.int32) - BIAS for s in (self.key_scales, self.value_scales))
        k = torch.ldexp(self.keys.float().view(pages, g, -1, BLOCK, d), ke[..., None, None])
        v = torch.ldexp(self.values.float().view(pages, g, d, -1, BLOCK), ve[:, :, None, :, None])
        return k.view(self.keys.shape).to(self.dtype), v.view(self.values.shape).to(self.dtype)


def _checked(what: str, pool: Fp8Pool, step: PagedStep) -> None:
    """The step's requests hold pages of this pool."""
    if not step.filled:
        raise ValueError("the step is empty: page_tables fills it")
    if step.state.page != pool.shape[2]:
        raise ValueError(f"{what}: the step is for pages of {step.state.page} positions, the pool has {pool.shape[2]}")
    if pool.shape[0] < step.state.free.numel():
        raise ValueError(f"the pool has {pool.shape[0]} pages, the page tables give out {step.state.free.numel()}")


def _page_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t[0].numel()


def rotary_paged_write_fp8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                           pool: Fp8Pool, step: PagedStep, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary on the step's packed rows ``q [rows, heads*d]`` and ``k [rows,
    kv_heads*d]``, and ``k`` and ``v`` into their slots of the pool; the rotated
    q (in ``out``, which may be ``q``, or a new tensor).

    ``cos`` and ``sin`` as for ``rotary_paged_write``; keys and values are fp32
    numbers rounded once, to the nearest code.  The exponent of a block that
    gets rows is the least one with ``max|new rows| <= 448 * 2**e`` (in bfloat16
    from -117 to 120, in float16 from -15 to 8; codes of the largest stop at
    240), or the one it has, where that is larger and the block holds earlier
    rows.  Infinities and NaN, and in float16 what rounds to infinity, are
    written as NaN and do not count.  Rows without a slot are rotated and not
    written.  Rows that replace others of their block (rejected drafts, a step
    that is run again) leave its exponent as high as those made it.  One write
    at a time may change a step's requests.
    """
    done = _ffi.calls().paged_write8(q, k, v, cos, sin, pool.keys, pool.values, pool.key_scales, pool.value_scales, pool._code,
                                     step._native, step.filled, out)
    if done is not None:
        return done if out is None else out
    what = "rotary_paged_write_fp8"
    cached = (pool.keys, pool.values, pool.key_scales, pool.value_scales)
    dev = _on_gpu(what, q, k, v, cos, sin, *cached, step.row_indptr)
    _untraced(what)
    _no_grad(what, q, k, v, cos, sin)
    _no_tangent(what, q, k, v, cos, sin)
    _checked(what, pool, step)
    pages, kv_heads, page, d = pool.shape
    rows, dt = step.rows, pool.dtype
    if q.dim() != 2 or q.shape[1] == 0 or q.shape[1] % d:
        raise ValueError(f"q must be [{rows}, heads * {d}], got {tuple(q.shape)}")
    heads = q.shape[1] // d
    _rows("q", q, rows, heads * d, dt)
    _rows("k", k, rows, kv_heads * d, dt)
    _rows("v", v, rows, kv_heads * d, dt)
    cos, sin = (t[:, 0] if t.dim() == 3 and t.shape[1] == 1 else t for t in (cos, sin))
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dim() != 2 or t.shape[0] not in (1, rows) or t.shape[1] != d or t.stride(1) != 1 or t.dtype not in (dt, torch.float32):
            raise ValueError(f"{name} must be [{rows} or 1, {d}] {dt} or float32, got {tuple(t.shape)} {t.dtype}")
    rot_stride = [0 if t.shape[0] == 1 else t.stride(0) for t in (cos, sin)]
    if cos.dtype != sin.dtype or rot_stride[0] != rot_stride[1]:
        raise ValueError("cos and sin must have one dtype and row stride")
    written = cached if out is None else (*cached, out)
    _writes(what, *written)
    if out is None:
        out = torch.empty((rows, heads * d), dtype=dt, device=dev)
    else:
        _on_gpu(what, q, out)
        _rows("out", out, rows, heads * d, dt)
    if rows == 0:
        return out
    stride = lambda t: t.stride(0) if rows > 1 else t.shape[1]  # noqa: E731
    with _guard(dev):
        rc = _ffi.lib().mlora_rotary_paged_write_fp8(
            q.data_ptr(), stride(q), k.data_ptr(), stride(k), v.data_ptr(), stride(v), cos.data_ptr(), sin.data_ptr(),
            rot_stride[0], _ffi.dtype_code(cos.dtype), step.slots.data_ptr(), rows, heads, kv_heads, d, pool.keys.data_ptr(),
            _page_stride(pool.keys), pool.values.data_ptr(), _page_stride(pool.values), pool.key_scales.data_ptr(),
            pool.value_scales.data_ptr(), pages, page, out.data_ptr(), stride(out), pool._code, _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_rotary_paged_write_fp8")
    torch.autograd.graph.increment_version(written)
    return out


def paged_attention_fp8(q: torch.Tensor, pool: Fp8Pool, step: PagedStep, scale: float,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the step's packed rows ``q [rows, heads*d]`` over
    their requests' pages of the pool, ``[rows, heads*d]``: ``paged_attention``
    over ``pool.dequantize()``, with the same rules for rows, steps and ``out``."""
    if not step.filled:
        raise ValueError("the step is empty: page_tables fills it")
    done = _ffi.calls().paged_attention8(q, pool.keys, pool.values, pool.key_scales, pool.value_scales, pool._code, step._native,
                                         scale, out)
    if done is not None:
        return done if out is None else out
    what = "paged_attention_fp8"
    dev = _on_gpu(what, q, pool.keys, step.row_indptr)
    _untraced(what)
    _no_grad(what, q, pool.keys, pool.values)
    _no_tangent(what, q, pool.keys, pool.values)
    _checked(what, pool, step)
    if not step.has_plan:
        raise ValueError("the step has no work list: give page_tables the heads")
    pages, kv_heads, page, d = pool.shape
    if (kv_heads, d) != (step.kv_heads, step.head_dim):
        raise ValueError(f"the step is for {step.kv_heads} key heads of {step.head_dim}, the pool has {kv_heads} of {d}")
    dt, width = pool.dtype, step.heads * d
    _rows("q", q, step.rows, width, dt)
    if step.rows > 1 and q.stride(0) % 8 or q.data_ptr() % 16:
        q = q.contiguous() if not q.is_contiguous() else q.clone()
    given = out is not None
    if given:
        _on_gpu(what, q, out)
        _writes(what, out)
        _rows("out", out, step.rows, width, dt)
    else:
        out = torch.empty((step.rows, width), dtype=dt, device=dev)
    stride = lambda t: t.stride(0) if step.rows > 1 else width  # noqa: E731
    with _guard(dev):
        rc = _ffi.lib().mlora_paged_attention_fp8(
            q.data_ptr(), stride(q), pool.keys.data_ptr(), _page_stride(pool.keys), pool.values.data_ptr(),
            _page_stride(pool.values), pool.key_scales.data_ptr(), pool.value_scales.data_ptr(), ctypes.byref(step.state._c),
            ctypes.byref(step._c), out.data_ptr(), stride(out), step.heads, kv_heads, d, float(scale), pool._code,
            _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_paged_attention_fp8")
    if given:
        torch.autograd.graph.increment_version(out)
    return out
