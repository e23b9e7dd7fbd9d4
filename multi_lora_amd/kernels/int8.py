"""Products of 16-bit activations with 8-bit weights, on the HIP kernels.

``quantize_rows`` turns every row of a matrix into 8-bit integers and one fp32
scale; ``int8_matmul`` multiplies two such matrices (a scale for each token,
and for each output channel), ``int8_linear`` quantises its activations on the
way.  ``layers.Int8Linear`` is the module over it, ``layers.quantize_base``
puts it in a model's place of its linear layers, beneath the adapters.

A row's scale is ``max|x| / 127``, its codes ``round(x / scale)``, ties to
even.  Sums of products are exact, so a result differs from that of exact
arithmetic on the codes only by its fp32 scaling and one rounding, and repeats
bit for bit.  Results are float16 or bfloat16.  There is no CPU path and no
derivative in either mode: inputs that ask for one are refused, and so are
calls under a trace, which would not see them.

No counterpart in the reference, whose base products are the model's own
(multi_lora/layers.py:42-88).
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from .. import _ffi
from .paged import _DTYPES, _guard, _no_grad, _no_tangent, _on_gpu, _untraced, _writes

PAD = 128        # columns of codes come in multiples of it
BAND = 16        # rows, too
MAX_K = (1 << 17) - 1  # longer sums of products could leave 32 bits
MAX_ROWS = (1 << 31) - 1  # the launches count rows in 32 bits


def _code_shape(rows: int, k: int):
    return (-(-k // PAD) * (PAD // 64), -(-rows // BAND), 4, BAND, 16)


@dataclass(frozen=True)
class Int8Rows:
    """Quantised rows ``[rows, k]``: 8-bit ``codes`` and ``scales [rows]``.  Row
    ``r`` stands for ``to_rows()[r] * scales[r]``.

    Codes lie in the order in which the matrix units take them, ``[k / 64,
    rows / 16, 4, 16, 16]`` (rounded up; ``k`` to a multiple of 128, zeros behind
    it): ``codes[e // 64, r // 16, e // 16 % 4, r % 16, e % 16]`` is column ``e``
    of row ``r``, and what the last rows' blocks hold behind them does not
    matter.  A slice of the second dimension is one, too.
    """

    codes: torch.Tensor   # int8
    scales: torch.Tensor  # float32
    k: int

    def __post_init__(self) -> None:
        c, s = self.codes, self.scales
        if not 1 <= self.k <= MAX_K:
            raise ValueError(f"rows of 1 to {MAX_K} elements, got {self.k}")
        if s.dtype != torch.float32 or s.dim() != 1 or not s.is_contiguous():
            raise ValueError(f"scales must be a contiguous float32 tensor of a number a row, got {tuple(s.shape)} {s.dtype}")
        if s.shape[0] > MAX_ROWS:
            raise ValueError(f"at most {MAX_ROWS} rows, got {s.shape[0]}")
        shape = _code_shape(s.shape[0], self.k)
        if (c.dtype != torch.int8 or tuple(c.shape) != shape or not c[0].is_contiguous() or c.data_ptr() % 16 or c.stride(0) % 16
                or c.stride(0) < shape[1] * 1024):
            raise ValueError(f"codes must be int8 of shape {shape} with contiguous blocks at multiples of 16 bytes, got "
                             f"{tuple(c.shape)} {c.dtype}")
        if s.device != c.device:
            raise ValueError(f"codes on {c.device}, scales on {s.device}")

    @property
    def shape(self):
        """``(rows, k)``."""
        return torch.Size((self.scales.shape[0], self.k))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor) -> "Int8Rows":
        """Rows quantised elsewhere: ``codes [rows, k]`` int8 and ``scales [rows]``; copied into the layout here."""
        if codes.dtype != torch.int8 or codes.dim() != 2:
            raise ValueError(f"codes must be int8 [rows, k], got {tuple(codes.shape)} {codes.dtype}")
        rows, k = codes.shape
        if not 1 <= k <= MAX_K:
            raise ValueError(f"rows of 1 to {MAX_K} elements, got {k}")
        blocks, bands = _code_shape(rows, k)[:2]
        padded = torch.zeros((bands * BAND, blocks * 64), dtype=torch.int8, device=codes.device)
        padded[:rows, :k] = codes
        padded = padded.view(bands, BAND, blocks, 4, 16).permute(2, 0, 3, 1, 4).contiguous()
        return cls(padded, scales.to(torch.float32).contiguous(), k)

    def to_rows(self) -> torch.Tensor:
        """The codes as a matrix, int8 ``[rows, k]``."""
        blocks, bands = self.codes.shape[:2]
        return self.codes.permute(1, 3, 0, 2, 4).reshape(bands * BAND, blocks * 64)[:self.shape[0], :self.k]

    def rows(self, start: int, end: int) -> "Int8Rows":
        """Rows ``[start, end)``: a view, where ``start`` is a multiple of 16, otherwise a copy."""
        start, end, _ = slice(start, end).indices(self.shape[0])
        end = max(start, end)
        if start % BAND == 0:
            return Int8Rows(self.codes[:, start // BAND:-(-end // BAND)], self.scales[start:end], self.k)
        return Int8Rows.from_codes(self.to_rows()[start:end], self.scales[start:end])

    @classmethod
    def cat(cls, parts: Sequence["Int8Rows"]) -> "Int8Rows":
        """The rows of several, one after the other."""
        if len({p.k for p in parts}) != 1:
            raise ValueError(f"rows of different lengths {[p.k for p in parts]}")
        scales = torch.cat([p.scales for p in parts])
        if all(p.shape[0] % BAND == 0 for p in parts[:-1]):
            return cls(torch.cat([p.codes for p in parts], 1), scales, parts[0].k)
        return cls.from_codes(torch.cat([p.to_rows() for p in parts]), scales)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the codes stand for, ``[rows, k]``."""
        return (self.to_rows().float() * self.scales[:, None]).to(dtype)


def _matrix(what: str, t: torch.Tensor, dtypes) -> None:
    if t.dim() != 2 or t.dtype not in dtypes or (t.numel() > 0 and t.stride(1) != 1):
        names = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        raise ValueError(f"{what} must be 2-D {names} with contiguous rows, got {tuple(t.shape)} {t.dtype}")
    if t.shape[0] > MAX_ROWS:
        raise ValueError(f"{what}: at most {MAX_ROWS} rows, got {t.shape[0]}")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: the rows overlap")


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two matrices share memory; columns of one buffer side by side do not."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    size, (sa, sb) = a.element_size(), (_stride(a), _stride(b))
    pa, pb = a.data_ptr(), b.data_ptr()
    ends = [p + ((t.shape[0] - 1) * s + t.shape[1]) * size for p, t, s in ((pa, a, sa), (pb, b, sb))]
    if ends[0] <= pb or ends[1] <= pa:
        return False
    apart = (pb - pa) // size % sa
    return sa != sb or apart < a.shape[1] or apart + b.shape[1] > sa


def quantize_rows(x: torch.Tensor) -> Int8Rows:
    """``x [rows, k]`` (float32, float16 or bfloat16) as 8-bit integers with a scale for each row.

    The maximum counts as at least ``2**-100``.  A row with an infinity or a
    NaN has a NaN scale (and a product with it a NaN result).  Codes of 16-bit
    rows are those of exact arithmetic; of float32 rows, those of fp32
    arithmetic, which may round a quotient next to halfway the other way.
    """
    dev = _on_gpu("quantize_rows", x)
    _untraced("quantize_rows")
    _no_grad("quantize_rows", x)
    _no_tangent("quantize_rows", x)
    _matrix("x", x, (torch.float32, *_DTYPES))
    rows, k = x.shape
    if not 1 <= k <= MAX_K:
        raise ValueError(f"rows of 1 to {MAX_K} elements, got {k}")
    codes = torch.empty(_code_shape(rows, k), dtype=torch.int8, device=dev)
    scales = torch.empty(rows, dtype=torch.float32, device=dev)
    with _guard(dev):
        rc = _ffi.lib().mlora_quantize_rows(x.data_ptr(), _stride(x), rows, k, codes.data_ptr(), scales.data_ptr(),
                                            _ffi.dtype_code(x.dtype), _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_quantize_rows")
    return Int8Rows(codes, scales, k)


def _result(what: str, rows: int, weight: Int8Rows, bias: Optional[torch.Tensor], out: Optional[torch.Tensor],
            dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """The checked or new output, and the bias checked."""
    n = weight.shape[0]
    if bias is not None:
        _on_gpu(what, weight.codes, bias)
        _no_grad(what, bias)
        _no_tangent(what, bias)
        if tuple(bias.shape) != (n,) or bias.dtype != dtype or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous {dtype} tensor of {n} numbers, got {tuple(bias.shape)} {bias.dtype}")
    if out is None:
        return torch.empty((rows, n), dtype=dtype, device=dev)
    _on_gpu(what, weight.codes, out)
    _writes(what, out)
    _no_tangent(what, out)
    _matrix("out", out, (dtype,))
    if tuple(out.shape) != (rows, n):
        raise ValueError(f"out must be [{rows}, {n}], got {tuple(out.shape)}")
    return out


def _address(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def int8_matmul(a: Int8Rows, b: Int8Rows, dtype: torch.dtype, bias: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a [m, k] @ b [n, k].T + bias`` of quantised rows, ``[m, n]`` in ``dtype`` (float16 or bfloat16; in ``out``
    if given, which may be a column slice of a wider tensor)."""
    dev = _on_gpu("int8_matmul", a.codes, b.codes)
    _untraced("int8_matmul")
    _no_grad("int8_matmul", a.scales, b.scales)
    _no_tangent("int8_matmul", a.scales, b.scales)
    if a.k != b.k:
        raise ValueError(f"rows of {a.k} and of {b.k} elements")
    if dtype not in _DTYPES:
        raise ValueError(f"int8_matmul: float16 or bfloat16, got {dtype}")
    m, n = a.shape[0], b.shape[0]
    given = out is not None
    out = _result("int8_matmul", m, b, bias, out, dtype, dev)
    with _guard(dev):
        rc = _ffi.lib().mlora_int8_matmul(a.codes.data_ptr(), a.codes.stride(0), a.scales.data_ptr(), m, b.codes.data_ptr(),
                                          b.codes.stride(0), b.scales.data_ptr(), n, a.k, _address(bias), out.data_ptr(),
                                          _stride(out), _ffi.dtype_code(dtype), _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_int8_matmul")
    if given:
        torch.autograd.graph.increment_version(out)
    return out


def int8_linear(x: torch.Tensor, weight: Int8Rows, bias: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [rows, k] @ weight.T + bias`` with the rows of ``x`` (float16 or bfloat16) quantised as ``quantize_rows``
    does; ``[rows, n]`` in x's type (in ``out`` if given, which may be a column slice of a wider tensor, and must not
    overlap ``x``).  A row with an infinity or a NaN gives NaN."""
    # The ordinary call, checked and launched natively; what it does not take (None) runs, or raises, below.
    done = _ffi.calls().int8_linear(x, weight.codes, weight.scales, weight.k, bias, out)
    if done is not None:
        return done if out is None else out
    dev = _on_gpu("int8_linear", x, weight.codes)
    _untraced("int8_linear")
    _no_grad("int8_linear", x, weight.scales)
    _no_tangent("int8_linear", x, weight.scales)
    _matrix("x", x, _DTYPES)
    rows, k = x.shape
    if k != weight.k:
        raise ValueError(f"x has rows of {k} elements, the weight of {weight.k}")
    given = out is not None
    out = _result("int8_linear", rows, weight, bias, out, x.dtype, dev)
    if given and _overlap(x, out):
        raise ValueError("int8_linear: out overlaps x")
    lib = _ffi.lib()
    need = lib.mlora_int8_linear_workspace_bytes(rows, k)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _guard(dev):
        rc = lib.mlora_int8_linear(x.data_ptr(), _stride(x), rows, weight.codes.data_ptr(), weight.codes.stride(0),
                                   weight.scales.data_ptr(), weight.shape[0], k, _address(bias), out.data_ptr(), _stride(out),
                                   _ffi.dtype_code(x.dtype), _address(ws), need, _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_int8_linear")
    if given:
        torch.autograd.graph.increment_version(out)
    return out
