"""A KV cache in pages that ragged requests share, on the HIP kernels.

``page_tables`` turns a step's request lengths into page tables, positions and
cache slots of its packed rows, and the work list of its attention;
``rotary_paged_write`` rotates q and k and writes k and v into their slots;
``paged_attention`` attends every row causally over its request's pages;
``verify_drafts`` checks drafted tokens against the target's probabilities.
The lengths live on the device and the host gives bounds only, so a step over
resident tensors can be captured in a HIP graph and replayed.

Pools of one layer: keys ``[num_pages, kv_heads, page, d]`` and values
``[num_pages, kv_heads, d, page]`` (transposed inside a page, so that a chunk
of eight positions is one load of the second product's operand).  Data in
float16 or bfloat16, ``d`` 64 or 128, pages of a power of two positions from 8
to 1024.  There is no CPU path and no derivative in either mode: inputs that ask
for one are refused, and so are calls under a trace, which would not see them.

No counterpart in the reference, whose decode runs over
``transformers.StaticCache`` (multi_lora/graph_decode.py:23-111).
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext
from dataclasses import dataclass, field
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from .. import _ffi

_DTYPES = (torch.float16, torch.bfloat16)


def _on_gpu(what: str, *tensors: torch.Tensor) -> torch.device:
    first = tensors[0].device
    if first.type != "cuda":
        raise RuntimeError(f"{what}: tensors must be on a ROCm GPU (got {first}); the HIP path has no CPU fallback")
    for t in tensors:
        if t.device != first:
            raise ValueError(f"{what}: tensors on {t.device} and {first}")
    return first


def _untraced(what: str) -> None:
    """The launch goes past torch: a trace would keep this call's result as a constant."""
    if torch.jit.is_tracing() or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise RuntimeError(f"{what} is not a torch operation and cannot be traced")


def _no_tangent(what: str, *tensors: torch.Tensor) -> None:
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative; call it on tensors without tangents")


def _no_grad(what: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward pass; call it under torch.no_grad() or on detached tensors")


def _writes(what: str, *tensors: torch.Tensor) -> None:
    """Tensors that a call is going to write."""
    _no_grad(what, *tensors)
    if any(t.is_inference() for t in tensors) and not torch.is_inference_mode_enabled():
        raise RuntimeError(f"{what} writes in place: inference tensors need inference mode")


def _guard(device: torch.device):
    """A launch goes to the current device."""
    return nullcontext() if device.index in (None, torch.cuda.current_device()) else torch.cuda.device(device)


def _i32(what: str, t: torch.Tensor, *shape: int) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape} (got {t.dtype} {tuple(t.shape)})")


@dataclass(frozen=True)
class PageState:
    """Which request holds which pages, on the device; ``page_tables`` changes
    it in place.  Request ``i`` holds ``table[i, :held[i]]``;
    ``free[:counts[0]]`` are the pages that none holds; ``counts[1]`` is how
    many pages the last call could not give."""

    table: torch.Tensor   # [n, width] int32
    held: torch.Tensor    # [n] int32
    free: torch.Tensor    # [num_pages] int32
    counts: torch.Tensor  # [2] int32
    page: int
    _c: _ffi.Pages = field(init=False, repr=False, compare=False)

    def __post_init__(self) -> None:
        if self.table.dim() != 2 or self.table.dtype != torch.int32 or (self.table.numel() > 0 and self.table.stride(1) != 1):
            raise ValueError("table must be an int32 tensor [n, width] with contiguous rows")
        n, width = self.table.shape
        if n > 1 and self.table.stride(0) < width:
            raise ValueError("the table's rows overlap")
        _i32("held", self.held, n)
        _i32("free", self.free, self.free.numel())
        _i32("counts", self.counts, 2)
        if any(t.device != self.table.device for t in (self.held, self.free, self.counts)):
            raise ValueError("table, held, free and counts must be on one device")
        page = int(self.page)
        if not 8 <= page <= 1024 or page & (page - 1):
            raise ValueError(f"pages of a power of two positions from 8 to 1024, got {page}")
        stride = self.table.stride(0) if n > 1 else width
        object.__setattr__(self, "_c", _ffi.Pages(self.table.data_ptr(), stride, self.held.data_ptr(), self.free.data_ptr(),
                                                  self.counts.data_ptr(), n, width, self.free.numel(), page))

    @classmethod
    def new(cls, seqs: int, max_len: int, num_pages: int, page: int, device) -> "PageState":
        """``seqs`` requests of up to ``max_len`` positions that hold nothing, and ``num_pages`` free pages."""
        i32 = dict(dtype=torch.int32, device=device)
        return cls(table=torch.full((seqs, -(-max_len // page)), -1, **i32), held=torch.zeros(seqs, **i32),
                   free=torch.arange(num_pages - 1, -1, -1, **i32),
                   counts=torch.tensor([num_pages, 0], **i32), page=page)


@lru_cache(maxsize=256)
def _step_sizes(n: int, rows: int, max_new: int, max_kv: int, heads: Optional[int], kv_heads: Optional[int],
                head_dim: Optional[int]) -> Tuple[int, int, int]:
    """(int32 words of scratch, of plan, bytes of workspace) of a step."""
    lib = _ffi.lib()
    scratch = lib.mlora_page_tables_scratch(n)
    if heads is None:
        return scratch, 0, 0
    pb, wb = ctypes.c_size_t(), ctypes.c_size_t()
    rc = lib.mlora_paged_step_bytes(n, rows, max_new, max_kv, heads, kv_heads, head_dim, ctypes.byref(pb), ctypes.byref(wb))
    _ffi.check(rc, "mlora_paged_step_bytes")
    return scratch, pb.value // 4, wb.value


class PagedStep:
    """The packed rows of one step: request ``i`` has rows ``[row_indptr[i],
    row_indptr[i + 1])``, the last of its ``kv_lens[i]`` positions.  Filled by
    ``page_tables``; with ``heads``, it carries the attention's work list and
    the workspace of its split ranges, so steps whose attention may overlap in
    time (on different streams) need to be different ``PagedStep``s, kept until
    those streams are done with them.

    ``row_indptr [n + 1]``, ``kv_lens [n]``, ``positions [rows]`` and ``slots
    [rows]`` (page * page size + offset; -1: no place) are int32 tensors.
    """

    __slots__ = ("state", "rows", "max_new", "heads", "kv_heads", "head_dim", "has_plan", "filled", "_ints", "_ends",
                 "_workspace", "_c", "_native")

    def __init__(self, state: PageState, rows: int, max_new: int, heads: Optional[int] = None,
                 kv_heads: Optional[int] = None, head_dim: Optional[int] = None) -> None:
        """Room for ``rows`` packed rows of at most ``max_new`` new tokens a request."""
        if rows < 0 or max_new < 0:
            raise ValueError(f"rows {rows}, max_new {max_new}")
        self.has_plan = heads is not None
        if not self.has_plan == (kv_heads is not None) == (head_dim is not None):
            raise ValueError("heads, kv_heads and head_dim are given together")
        n, width = state.table.shape
        scratch, plan, ws = _step_sizes(n, rows, max_new, width * state.page, heads, kv_heads, head_dim)
        dev = state.table.device
        self.state, self.rows, self.max_new = state, rows, max_new
        self.filled = False  # by page_tables
        self.heads, self.kv_heads, self.head_dim = heads or 0, kv_heads or 0, head_dim or 0
        # One buffer: the tensors below, the tables' scratch, the plan.
        self._ends = ends = (n + 1, 2 * n + 1, 2 * n + 1 + rows, 2 * n + 1 + 2 * rows)
        self._ints = ints = torch.empty(ends[3] + scratch + plan, dtype=torch.int32, device=dev)
        self._workspace = torch.empty(ws, dtype=torch.uint8, device=dev) if ws else None
        p = ints.data_ptr()
        at = p + 4 * (ends[3] + scratch)
        self._c = _ffi.PagedStep(p, p + 4 * ends[0], p + 4 * ends[1], p + 4 * ends[2], at if self.has_plan else None,
                                 self._workspace.data_ptr() if ws else None, 4 * plan, ws, rows, max_new)
        self._native = (ctypes.addressof(state._c), ctypes.addressof(self._c), p + 4 * ends[3], self.heads, self.kv_heads,
                        self.head_dim, -1 if dev.index is None else dev.index)

    @property
    def row_indptr(self) -> torch.Tensor:
        return self._ints[:self._ends[0]]

    @property
    def kv_lens(self) -> torch.Tensor:
        return self._ints[self._ends[0]:self._ends[1]]

    @property
    def positions(self) -> torch.Tensor:
        return self._ints[self._ends[1]:self._ends[2]]

    @property
    def slots(self) -> torch.Tensor:
        return self._ints[self._ends[2]:self._ends[3]]


def page_tables(state: PageState, start_lens: torch.Tensor, new_lens: torch.Tensor, *, rows: Optional[int] = None,
                max_new: Optional[int] = None, heads: Optional[int] = None, kv_heads: Optional[int] = None,
                head_dim: Optional[int] = None, step: Optional[PagedStep] = None) -> PagedStep:
    """Pages, slots and positions of a step in which request ``i`` keeps
    ``start_lens[i]`` cached positions and gets ``new_lens[i]`` tokens (int32
    tensors on the device).

    Requests take the pages that they lack and give back those past their new
    length (0 and 0: a request that is done; a smaller start: tokens taken
    back), in request order; ``state`` changes in place.  A page that the pool
    cannot give is counted in ``state.counts[1]``; its tokens have slot -1 and
    are not written, and this step's rows that would attend to it are NaN.
    Such tokens are not cached: the next call, which may get the page, keeps at
    most ``torch.minimum(step.kv_lens, state.held * state.page)`` positions.

    ``rows`` (packed rows, at least the sum of the new lengths) and ``max_new``
    (at least each of them) are the host's bounds: a longer new length counts
    as ``max_new``, requests that the rows do not hold get fewer or none.  Rows
    behind the last request's get position 0 and slot -1.  With ``heads``, ``kv_heads`` and
    ``head_dim`` the step carries what ``paged_attention`` needs.  ``step``:
    one to fill again in place (its bounds and heads hold), as a captured step
    does (``start_lens`` may be its ``kv_lens``); otherwise a new one is
    returned.  Calls on one state are made in order, on one stream or with the
    streams made to wait.
    """
    if step is None:
        if rows is None or max_new is None:
            raise ValueError("page_tables needs rows and max_new, or a step to fill")
        step = PagedStep(state, rows, max_new, heads, kv_heads, head_dim)
    elif any(v is not None for v in (rows, max_new, heads, kv_heads, head_dim)):
        raise ValueError("a step to fill again keeps its own bounds and heads")
    elif step.state is not state:
        raise ValueError("the step belongs to another PageState")
    if _ffi.calls().page_tables(step._native, start_lens, new_lens):
        step.filled = True
        return step
    dev = _on_gpu("page_tables", state.table, start_lens, new_lens)
    _untraced("page_tables")
    n = state.table.shape[0]
    _i32("start_lens", start_lens, n)
    _i32("new_lens", new_lens, n)
    with _guard(dev):
        rc = _ffi.lib().mlora_page_tables(ctypes.byref(state._c), start_lens.data_ptr(), new_lens.data_ptr(),
                                          ctypes.byref(step._c), step.heads, step.kv_heads, step.head_dim,
                                          step._native[2], _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_page_tables")
    step.filled = True
    return step


def _pool(what: str, keys: torch.Tensor, values: torch.Tensor) -> Tuple[int, int, int, int]:
    """(num_pages, kv_heads, page, d) of one layer's pools."""
    if keys.dim() != 4 or values.dim() != 4:
        raise ValueError(f"{what}: keys [num_pages, kv_heads, page, d] and values [num_pages, kv_heads, d, page]")
    pages, kv_heads, page, d = keys.shape
    if values.shape != (pages, kv_heads, d, page) or values.dtype != keys.dtype:
        raise ValueError(f"{what}: keys {tuple(keys.shape)} {keys.dtype}, values {tuple(values.shape)} {values.dtype}")
    if keys.dtype not in _DTYPES:
        raise ValueError(f"{what}: float16 or bfloat16, got {keys.dtype}")
    if pages == 0 or not keys[0].is_contiguous() or not values[0].is_contiguous():
        raise ValueError(f"{what}: every page must be contiguous, and there must be one")
    return pages, kv_heads, page, d


def _rows(what: str, t: torch.Tensor, rows: int, width: int, dtype: torch.dtype) -> None:
    if t.dim() != 2 or t.shape != (rows, width) or t.dtype != dtype or (t.numel() > 0 and t.stride(1) != 1):
        raise ValueError(f"{what} must be [{rows}, {width}] {dtype} with contiguous rows, got {tuple(t.shape)} {t.dtype}")


def rotary_paged_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                       keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary on the packed rows ``q [rows, heads*d]`` and ``k [rows,
    kv_heads*d]``, and ``k`` and ``v`` into their ``slots`` of the pools; the
    rotated q (in ``out``, which may be ``q``, or a new tensor).

    ``cos`` and the signed ``sin`` are ``decoder.Rotary``'s tables (``[rows or
    1, d]`` or ``[rows or 1, 1, d]``, the data type or float32): ``x * cos +
    roll(x, d/2) * sin`` in fp32, rounded once.  Rows with a slot outside the
    pool are rotated and not written.  The slots of one call must differ.
    """
    # The ordinary call, checked and launched natively; what it does not take
    # (None) runs, or raises, below.  So in the functions after this one.
    done = _ffi.calls().paged_write(q, k, v, cos, sin, keys, values, slots, out)
    if done is not None:
        return done if out is None else out
    dev = _on_gpu("rotary_paged_write", q, k, v, cos, sin, keys, values, slots)
    _untraced("rotary_paged_write")
    _no_grad("rotary_paged_write", q, k, v, cos, sin, keys, values)
    _no_tangent("rotary_paged_write", q, k, v, cos, sin, keys, values)
    pages, kv_heads, page, d = _pool("rotary_paged_write", keys, values)
    rows = q.shape[0] if q.dim() == 2 else -1
    if rows < 0 or q.shape[1] == 0 or q.shape[1] % d:
        raise ValueError(f"q must be [rows, heads * {d}], got {tuple(q.shape)}")
    heads = q.shape[1] // d
    dt = keys.dtype
    _rows("q", q, rows, heads * d, dt)
    _rows("k", k, rows, kv_heads * d, dt)
    _rows("v", v, rows, kv_heads * d, dt)
    _i32("slots", slots, rows)
    cos, sin = (t[:, 0] if t.dim() == 3 and t.shape[1] == 1 else t for t in (cos, sin))
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dim() != 2 or t.shape[0] not in (1, rows) or t.shape[1] != d or t.stride(1) != 1 or t.dtype not in (dt, torch.float32):
            raise ValueError(f"{name} must be [{rows} or 1, {d}] {dt} or float32, got {tuple(t.shape)} {t.dtype}")
    rot_stride = [0 if t.shape[0] == 1 else t.stride(0) for t in (cos, sin)]
    if cos.dtype != sin.dtype or rot_stride[0] != rot_stride[1]:
        raise ValueError("cos and sin must have one dtype and row stride")
    written = (keys, values) if out is None else (keys, values, out)
    _writes("rotary_paged_write", *written)
    if out is None:
        out = torch.empty((rows, heads * d), dtype=dt, device=dev)
    else:
        _on_gpu("rotary_paged_write", q, out)
        _rows("out", out, rows, heads * d, dt)
    if rows == 0:
        return out
    stride = lambda t: t.stride(0) if rows > 1 else t.shape[1]  # noqa: E731
    with _guard(dev):
        rc = _ffi.lib().mlora_rotary_paged_write(
            q.data_ptr(), stride(q), k.data_ptr(), stride(k), v.data_ptr(), stride(v), cos.data_ptr(), sin.data_ptr(),
            rot_stride[0], _ffi.dtype_code(cos.dtype), slots.data_ptr(), rows, heads, kv_heads, d, keys.data_ptr(),
            keys.stride(0) if pages > 1 else kv_heads * page * d, values.data_ptr(),
            values.stride(0) if pages > 1 else kv_heads * page * d, pages, page, out.data_ptr(), stride(out),
            _ffi.dtype_code(dt), _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_rotary_paged_write")
    torch.autograd.graph.increment_version(written)
    return out


def paged_attention(q: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, step: PagedStep, scale: float,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the step's packed rows ``q [rows, heads*d]`` over
    their requests' pages; ``[rows, heads*d]``.

    Row ``r`` of a request attends to the positions up to its own, the cached
    ones and those written in this step; query heads share key heads in order
    (``heads / kv_heads`` each).  ``step`` is ``page_tables``' of this step,
    made for these heads; one step serves every layer.  Sums are fp32 and the
    result is rounded once.  Rows behind the last request's are left as they
    were in ``out`` (undefined without one).  A step whose ``page_tables`` was
    only recorded holds a work list once the graph has run; before, the result
    is undefined.
    """
    if not step.filled:
        raise ValueError("the step is empty: page_tables fills it")
    done = _ffi.calls().paged_attention(q, keys, values, step._native, scale, out)
    if done is not None:
        return done if out is None else out
    dev = _on_gpu("paged_attention", q, keys, values, step.row_indptr)
    _untraced("paged_attention")
    _no_grad("paged_attention", q, keys, values)
    _no_tangent("paged_attention", q, keys, values)
    pages, kv_heads, page, d = _pool("paged_attention", keys, values)
    if not step.has_plan:
        raise ValueError("the step has no work list: give page_tables the heads")
    if (kv_heads, d, page) != (step.kv_heads, step.head_dim, step.state.page):
        raise ValueError(f"the step is for {step.kv_heads} key heads of {step.head_dim} and pages of {step.state.page}, the "
                         f"pool has {kv_heads}, {d} and {page}")
    dt = keys.dtype
    width = step.heads * d
    _rows("q", q, step.rows, width, dt)
    if pages < step.state.free.numel():
        raise ValueError(f"the pool has {pages} pages, the page tables give out {step.state.free.numel()}")
    if step.rows > 1 and q.stride(0) % 8 or q.data_ptr() % 16:
        q = q.contiguous() if not q.is_contiguous() else q.clone()
    given = out is not None
    if given:
        _on_gpu("paged_attention", q, out)
        _writes("paged_attention", out)
        _rows("out", out, step.rows, width, dt)
    else:
        out = torch.empty((step.rows, width), dtype=dt, device=dev)
    stride = lambda t: t.stride(0) if step.rows > 1 else width  # noqa: E731
    with _guard(dev):
        rc = _ffi.lib().mlora_paged_attention(
            q.data_ptr(), stride(q), keys.data_ptr(), keys.stride(0) if pages > 1 else kv_heads * page * d,
            values.data_ptr(), values.stride(0) if pages > 1 else kv_heads * page * d, ctypes.byref(step.state._c),
            ctypes.byref(step._c), out.data_ptr(), stride(out), step.heads, kv_heads, d, float(scale),
            _ffi.dtype_code(dt), _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_paged_attention")
    if given:
        torch.autograd.graph.increment_version(out)
    return out


def verify_drafts(target: torch.Tensor, draft: Optional[torch.Tensor], tokens: torch.Tensor, row_indptr: torch.Tensor,
                  accept: torch.Tensor, last: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Accepted drafts of each request and the token after them.

    Request ``i`` has rows ``[row_indptr[i], row_indptr[i + 1])`` of the
    target's probabilities ``target [rows, vocab]``: the distribution of the
    token after its last confirmed one, then after each of its drafts
    ``tokens[i, :k]`` (int64 ``[n, most]``; ``k`` is one less than its rows).
    ``draft [n, most, vocab]`` are the probabilities that the drafts were drawn
    from, None for drafts that were certain.  Draft ``j`` is accepted while
    ``accept[i, j] * draft[i, j, x] < target[row + j, x]``.  The next token is
    drawn with ``last[i]`` from ``max(target - draft, 0)`` of the first
    rejection, or from the row after the last draft: the lowest token whose
    cumulated mass exceeds ``last[i]`` times the total.  ``accept [n, most]``
    and ``last [n]`` are fp32 numbers in [0, 1).

    Returns ``accepted [n]`` (int32) and ``[n, most + 1]`` (int64): the accepted
    drafts, the next token, then -1.  A request without rows gets 0 and -1; a
    row without any mass, -1.  Probabilities are float32, float16 or bfloat16;
    all sums are fp64, so a draw differs from that of exact sums only where
    ``last[i]`` lies within about ``vocab * 2**-53`` of a column's border.
    """
    done = _ffi.calls().verify_drafts(target, draft, tokens, row_indptr, accept, last)
    if done is not None:
        return done
    given = [t for t in (target, draft, tokens, row_indptr, accept, last) if t is not None]
    dev = _on_gpu("verify_drafts", *given)
    _untraced("verify_drafts")
    if tokens.dim() != 2 or tokens.dtype != torch.int64 or (tokens.numel() > 0 and tokens.stride(1) != 1):
        raise ValueError("tokens must be int64 [n, most] with contiguous rows")
    n, most = tokens.shape
    _i32("row_indptr", row_indptr, n + 1)
    if target.dim() != 2 or target.shape[1] == 0 or (target.numel() > 0 and target.stride(1) != 1):
        raise ValueError("target must be [rows, vocab] with contiguous rows")
    rows, vocab = target.shape
    code = _ffi.dtype_code(target.dtype)
    if accept.shape != (n, most) or accept.dtype != torch.float32 or (accept.numel() > 0 and accept.stride(1) != 1):
        raise ValueError(f"accept must be float32 [{n}, {most}] with contiguous rows")
    if last.shape != (n,) or last.dtype != torch.float32 or not last.is_contiguous():
        raise ValueError(f"last must be a contiguous float32 tensor of {n} numbers")
    if draft is not None and (draft.shape != (n, most, vocab) or draft.dtype != target.dtype
                              or (draft.numel() > 0 and draft.stride(2) != 1)):
        raise ValueError(f"draft must be {target.dtype} [{n}, {most}, {vocab}] with contiguous rows")
    lib = _ffi.lib()
    accepted = torch.empty(n, dtype=torch.int32, device=dev)
    out = torch.empty((n, most + 1), dtype=torch.int64, device=dev)
    if n == 0:
        return accepted, out
    need = lib.mlora_verify_workspace_bytes(n, vocab)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    with _guard(dev):
        rc = lib.mlora_verify_drafts(
            target.data_ptr(), target.stride(0) if rows > 1 else vocab, rows,
            draft.data_ptr() if draft is not None else None, draft.stride(0) if draft is not None else 0,
            draft.stride(1) if draft is not None else 0, tokens.data_ptr(), tokens.stride(0), row_indptr.data_ptr(),
            accept.data_ptr(), accept.stride(0), last.data_ptr(), n, most, vocab, accepted.data_ptr(), out.data_ptr(),
            code, ws.data_ptr(), need, _ffi.stream_ptr(dev))
    _ffi.check(rc, "mlora_verify_drafts")
    return accepted, out
