"""HIP segment-LoRA kernels (export surface of multi_lora/kernels/__init__.py:3-7)."""

from .int8 import Int8Rows, int8_linear, int8_matmul, quantize_rows
from .lora_ops import (
    Workspace,
    sgemm_lora_a_fwd,
    sgemm_lora_a_multi_fwd,
    sgemm_lora_b_fwd,
    sgemm_lora_b_multi_fwd,
)
from .paged import PagedStep, PageState, page_tables, paged_attention, rotary_paged_write, verify_drafts
from .paged8 import Fp8Pool, paged_attention_fp8, rotary_paged_write_fp8
from .rmsnorm import fuse_rmsnorm, fused_add_rmsnorm, rmsnorm_fwd
from .scatter_bank import scatter_stage

__all__ = [
    "Workspace",
    "sgemm_lora_a_fwd",
    "sgemm_lora_b_fwd",
    "scatter_stage",
    "sgemm_lora_a_multi_fwd",
    "sgemm_lora_b_multi_fwd",
    "rmsnorm_fwd",
    "fuse_rmsnorm",
    "fused_add_rmsnorm",
    "PageState",
    "PagedStep",
    "page_tables",
    "rotary_paged_write",
    "paged_attention",
    "verify_drafts",
    "Fp8Pool",
    "rotary_paged_write_fp8",
    "paged_attention_fp8",
    "Int8Rows",
    "quantize_rows",
    "int8_matmul",
    "int8_linear",
]
