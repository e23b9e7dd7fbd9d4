"""LoRA-wrapped linear layers (mirrors multi_lora/layers.py:13-142).

``LinearWithLoRA`` computes the base GEMM and then lets the backend add
every segment's LoRA delta into the result in place; the result may be a
strided view (a column slice of a fused QKV output) and is never copied.
``QKVProjGroup`` fuses the q/k/v base GEMMs of one attention block in decode;
when the backend offers ``apply_lora_multi`` the three LoRA deltas are also
applied by one shrink (x read once) and one three-slice expand.

``Int8Linear`` is a linear layer whose weight is held in 8-bit integers
(``kernels.int8``); ``quantize_base`` puts it in place of a model's ``nn.Linear``
layers, wrapped ones too.  The adapters above stay as they are: a delta is
added to the layer's 16-bit result from its 16-bit input.  No counterpart in
the reference.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Sequence, Union

import torch
import torch.nn as nn
import torch.nn.functional as F

from .backend.base import LoRABackend
from .kernels.int8 import BAND, Int8Rows, int8_linear, quantize_rows

# Process-wide switch: when off, wrapped layers return the base output only.
LORA_ENABLED = True


def set_lora_enabled(enabled: bool) -> None:
    global LORA_ENABLED
    LORA_ENABLED = bool(enabled)


def lora_delta(x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: float, *, rank: int) -> torch.Tensor:
    """Closed form ``scaling * x @ A[:rank].T @ B[:, :rank].T`` (a test helper, not a kernel path)."""
    a = lora_a[:rank]
    b = lora_b[:, :rank]
    flat = x.reshape(-1, x.shape[-1])
    delta = (flat @ a.T @ b.T) * scaling
    return delta.reshape(*x.shape[:-1], b.shape[0])


class LinearWithLoRA(nn.Module):
    """``base_layer(x)`` plus the per-segment LoRA delta from the backend."""

    def __init__(self, base_layer: nn.Module) -> None:
        super().__init__()
        self.base_layer = base_layer
        self.backend: Optional[LoRABackend] = None
        self.A_buffer: Optional[torch.Tensor] = None
        self.B_buffer: Optional[torch.Tensor] = None
        self.qkv_group: Optional["QKVProjGroup"] = None
        self.qkv_slice: Optional[tuple] = None

    def set_lora_info(self, backend: LoRABackend, a_buffer: torch.Tensor, b_buffer: torch.Tensor) -> None:
        """Bind the step's backend and this module's slot stacks ``[K, r_max, in]`` / ``[K, out, r_max]``."""
        self.backend = backend
        self.A_buffer = a_buffer
        self.B_buffer = b_buffer

    def has_lora(self) -> bool:
        return LORA_ENABLED and self.backend is not None and self.A_buffer is not None and self.B_buffer is not None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if self.qkv_group is not None:
            return self.qkv_group.forward(self, x)
        return self.add_delta(x, self.base_layer(x))

    def add_delta(self, x: torch.Tensor, y_base: torch.Tensor) -> torch.Tensor:
        """Add the LoRA delta into ``y_base`` (possibly a strided view) and return it."""
        if not self.has_lora():
            return y_base
        x_flat = x.reshape(-1, x.shape[-1])
        y_flat = y_base.reshape(-1, y_base.shape[-1])
        y_flat = self.backend.apply_lora(x_flat, self.A_buffer, self.B_buffer, y_flat)
        return y_flat.reshape(y_base.shape)


def _packed(x: torch.Tensor) -> torch.Tensor:
    """``x [..., k]`` as rows that lie apart, each contiguous: what the kernels take (copied only if it is not)."""
    rows = x.reshape(-1, x.shape[-1])
    if rows.stride(1) != 1 or rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]:
        rows = rows.clone(memory_format=torch.contiguous_format)
    return rows


def _int8_product(x: torch.Tensor, weight: Int8Rows, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x [..., k] @ weight.T + bias``; under autocast x and bias are cast as those of ``F.linear`` are."""
    if torch.is_autocast_enabled("cuda") and x.is_floating_point() and x.dtype != torch.float64:
        dtype = torch.get_autocast_dtype("cuda")
        x, bias = x.to(dtype), None if bias is None else bias.to(dtype)
    return int8_linear(_packed(x), weight, bias).view(*x.shape[:-1], weight.shape[0])


class Int8Linear(nn.Module):
    """``y = x @ weight.T + bias`` for 16-bit ``x`` (under autocast also for
    float32), with the weight in 8-bit integers and a scale for each output
    channel, and x's rows quantised at every call.  GPU only; no gradients (a
    model that serves)."""

    def __init__(self, weight: Int8Rows, bias: Optional[torch.Tensor] = None) -> None:
        super().__init__()
        self.register_buffer("codes", None)
        self.register_buffer("scales", None)
        self.register_buffer("bias", None if bias is None else bias.detach())
        self.weight = weight

    @classmethod
    def from_linear(cls, layer: nn.Linear) -> "Int8Linear":
        """The layer with its weight quantised (on the GPU)."""
        return cls(quantize_rows(layer.weight.detach()), layer.bias).train(layer.training)

    @property
    def weight(self) -> Int8Rows:
        w = self._weight
        if w.codes is not self.codes or w.scales is not self.scales:  # buffers replaced (a state dict assigned)
            w = self._weight = Int8Rows(self.codes, self.scales, self.in_features)
        return w

    @weight.setter
    def weight(self, weight: Int8Rows) -> None:
        self.out_features, self.in_features = weight.shape
        self.codes, self.scales = weight.codes, weight.scales
        self._weight = weight

    def _apply(self, fn, recurse: bool = True):
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != scales.dtype:  # a change of the model's type is not one of the scales'
            self.scales = scales.to(self.scales.device)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return _int8_product(x, self.weight, self.bias)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def _in_bands(parts: Sequence[Int8Rows]) -> Int8Rows:
    """Their rows one after the other, each part in whole bands of its own, so that a part's blocks hold no other's rows:
    rows behind a part's last, up to a multiple of 16, have a scale of 0 (and products that nobody looks at)."""
    if len({p.k for p in parts}) != 1:
        raise ValueError(f"rows of different lengths {[p.k for p in parts]}")
    scales = torch.cat([F.pad(p.scales, (0, -p.shape[0] % BAND)) for p in parts])
    return Int8Rows(torch.cat([p.codes for p in parts], 1), scales, parts[0].k)


class QKVProjGroup:
    """One base GEMM and one multi-slice LoRA call for sibling projections
    that read the same input: q/k/v of an attention block
    (multi_lora/layers.py:91-142), or gate/up of an MLP.  Bias-free.

    Decode-shaped inputs (one row per sequence) always take the fused path,
    as in the reference.  With ``all_shapes`` every input does: prefill and
    mixed batches then read x once for all slices, in one library call.
    """

    def __init__(self, wrappers: List[LinearWithLoRA], all_shapes: bool = False) -> None:
        self.wrappers = list(wrappers)
        self._parts: List[tuple] = []  # 8-bit: codes and scales of each layer, views of the fused weight's
        self._join()
        for w in wrappers:
            w.qkv_group = self
        # One call's input (and its version), its result, and the projections that have not taken theirs.
        self._cached_x: Optional[torch.Tensor] = None
        self._cached_version: Optional[int] = None
        self._cached_out: Optional[torch.Tensor] = None
        self._waiting: set = set()
        self._delta_done = False
        self.all_shapes = all_shapes

    def _join(self) -> None:
        """The fused weight; each layer's becomes a view of it: no extra memory."""
        layers = [w.base_layer for w in self.wrappers]
        if any(m.bias is not None for m in layers):
            raise RuntimeError("QKV fusion requires bias=None")
        eight = isinstance(layers[0], Int8Linear)
        if any(isinstance(m, Int8Linear) != eight for m in layers):
            raise RuntimeError("fusion of 8-bit and 16-bit projections")
        # Where a projection's columns begin: one after the other, 8-bit ones in bands of rows of their own.
        step = BAND if eight else 1
        self.weight: Union[torch.Tensor, Int8Rows] = (
            _in_bands([m.weight for m in layers]) if eight else torch.cat([m.weight.detach() for m in layers], dim=0))
        col = 0
        for w, m in zip(self.wrappers, layers):
            width = int(m.weight.shape[0])
            m.weight = (self.weight.rows(col, col + width) if eight
                        else nn.Parameter(self.weight[col : col + width], requires_grad=False))
            w.qkv_slice = (col, col + width)
            col += -(-width // step) * step
        if eight:
            self._parts = [(m.codes, m.scales) for m in layers]

    def _follow(self) -> None:
        """8-bit: the fused weight again, where a layer or its buffers were replaced (a state dict assigned, a move)."""
        for w, (codes, scales) in zip(self.wrappers, self._parts):
            held = w.base_layer._buffers
            if held.get("codes") is not codes or held.get("scales") is not scales:
                with torch.inference_mode(False):
                    return self._join()

    def _multi_ready(self) -> bool:
        first = self.wrappers[0]
        return (
            all(w.has_lora() for w in self.wrappers)
            and all(w.backend is first.backend for w in self.wrappers)
            and hasattr(first.backend, "apply_lora_multi")
            and len({w.A_buffer.shape[1] for w in self.wrappers}) == 1
        )

    def _base(self, x: torch.Tensor) -> torch.Tensor:
        if isinstance(self.weight, Int8Rows):
            self._follow()
        if isinstance(self.weight, Int8Rows):
            return _int8_product(x, self.weight)
        return F.linear(x, self.weight)

    def forward(self, wrapper: LinearWithLoRA, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-2] != 1 and not self.all_shapes:
            return wrapper.add_delta(x, wrapper.base_layer(x))
        version = None if x.is_inference() else x._version
        if self._cached_x is not x or self._cached_version != version or wrapper not in self._waiting:
            self._cached_x = None  # if this call raises, the next one computes
            self._cached_out = self._base(x)
            self._delta_done = False
            if self._multi_ready():
                first = self.wrappers[0]
                x_flat = x.reshape(-1, x.shape[-1])
                out_flat = self._cached_out.reshape(-1, self._cached_out.shape[-1])
                first.backend.apply_lora_multi(
                    x_flat,
                    [w.A_buffer for w in self.wrappers],
                    [w.B_buffer for w in self.wrappers],
                    out_flat,
                    [w.qkv_slice[0] for w in self.wrappers],
                )
                self._delta_done = True
            self._cached_x, self._cached_version = x, version
            self._waiting = set(self.wrappers)
        start, end = wrapper.qkv_slice
        y = self._cached_out[..., start:end]
        self._waiting.discard(wrapper)
        if self._delta_done:
            return y
        return wrapper.add_delta(x, y)


QKV_LEAVES = ("q_proj", "k_proj", "v_proj")
GATE_UP_LEAVES = ("gate_proj", "up_proj")


def _fuse_siblings(wrappers: Dict[str, LinearWithLoRA], leaves, all_shapes: bool) -> int:
    """Group the wrappers named ``<parent>.<leaf>`` by parent; every parent
    holding all of ``leaves`` becomes one group, in ``leaves`` order."""
    blocks: Dict[str, Dict[str, LinearWithLoRA]] = {}
    for name, wrapper in wrappers.items():
        parent, dot, leaf = name.rpartition(".")
        if dot and leaf in leaves and wrapper.qkv_group is None:
            blocks.setdefault(parent, {})[leaf] = wrapper
    complete = [block for block in blocks.values() if len(block) == len(leaves)]
    for block in complete:
        QKVProjGroup([block[leaf] for leaf in leaves], all_shapes=all_shapes)
    return len(complete)


def fuse_qkv_projections(wrappers: Dict[str, LinearWithLoRA], all_shapes: bool = False) -> int:
    """Fuse the base GEMMs of every attention block whose q, k and v
    projections are all wrapped (multi_lora/layers.py:128-142); returns the
    number of blocks fused.  Wrappers are matched by their parent module's
    name, so ``...self_attn.q_proj`` joins ``...self_attn.k_proj``."""
    return _fuse_siblings(wrappers, QKV_LEAVES, all_shapes)


def fuse_gate_up_projections(wrappers: Dict[str, LinearWithLoRA], all_shapes: bool = True) -> int:
    """The same for every MLP whose gate and up projections are both wrapped:
    one base GEMM and one two-slice LoRA call over their shared input."""
    return _fuse_siblings(wrappers, GATE_UP_LEAVES, all_shapes)


# What a module calls besides its forward.
_HOOKS = ("_forward_pre_hooks", "_forward_hooks", "_backward_pre_hooks", "_backward_hooks", "_state_dict_pre_hooks",
          "_state_dict_hooks", "_load_state_dict_pre_hooks", "_load_state_dict_post_hooks")


def quantize_base(model: nn.Module, skip: Sequence[str] = ("lm_head",)) -> int:
    """Replace the model's ``nn.Linear`` layers (on the GPU), those beneath
    ``LinearWithLoRA`` too, by ``Int8Linear``; returns how many (one that
    stands in several places is one, there too).  Layers whose last name is in
    ``skip`` stay, and so does what is not a float16 or bfloat16 layer, or is of
    a class derived from ``nn.Linear``; a layer with hooks is refused before any
    is replaced.  Call it before projections are fused; adapters may be
    registered and layers wrapped before or after."""
    if type(model) is nn.Linear:
        raise ValueError("a layer cannot replace itself: Int8Linear.from_linear")
    for name, module in model.named_modules():
        if isinstance(module, LinearWithLoRA) and module.qkv_group is not None:
            raise RuntimeError(f"{name} is part of a fused group: quantise the base before fusing projections")
    places = []
    for name, module in model.named_modules(remove_duplicate=False):  # a layer in several places: each of them
        leaf = [part for part in name.split(".") if part != "base_layer"][-1:]
        if type(module) is not nn.Linear or (leaf and leaf[0] in skip):
            continue
        if module.weight.dtype not in (torch.float16, torch.bfloat16):
            continue
        if any(getattr(module, hooks) for hooks in _HOOKS) or "forward" in module.__dict__:
            raise RuntimeError(f"{name} has hooks, which would be lost with the layer: remove them, or skip it")
        places.append((name, module))
    replaced: Dict[nn.Module, Int8Linear] = {}
    for name, module in places:
        parent, _, child = name.rpartition(".")
        if module not in replaced:
            replaced[module] = Int8Linear.from_linear(module)
        setattr(model.get_submodule(parent) if parent else model, child, replaced[module])
    return len(replaced)
