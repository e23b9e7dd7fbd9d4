"""More rows than the launches of products in 8-bit integers can count (on tensors without storage)."""

import pytest
import torch

from multi_lora_amd.kernels import Int8Rows
from multi_lora_amd.kernels import int8

MANY = 2 ** 32 + 5  # 5 in 32 bits


def test_matrices_of_too_many_rows_are_refused():
    for rows in (2 ** 31, 2 ** 32, MANY):
        with pytest.raises(ValueError, match="at most"):
            int8._matrix("x", torch.empty((rows, 1), dtype=torch.bfloat16, device="meta"), (torch.bfloat16,))
    int8._matrix("x", torch.empty((2 ** 31 - 1, 1), dtype=torch.bfloat16, device="meta"), (torch.bfloat16,))


def test_quantised_rows_that_are_too_many_are_refused():
    codes = torch.empty((2, -(-MANY // 16), 4, 16, 16), dtype=torch.int8, device="meta")
    with pytest.raises(ValueError, match="at most"):
        Int8Rows(codes, torch.empty(MANY, device="meta"), 100)
