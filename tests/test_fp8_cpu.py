"""Wrapping stored fp8 codes: what is taken, what is refused."""

from __future__ import annotations

import pytest
import torch

from moss_image_b200.fp8 import FrozenFp8Linear


def _codes(rows: int, columns: int) -> torch.Tensor:
    return torch.zeros(rows, columns, dtype=torch.uint8).view(torch.float8_e4m3fn)


def test_a_strided_bias_is_made_dense():
    bias = torch.arange(40.0)[::2]
    module = FrozenFp8Linear.from_codes(_codes(20, 32), torch.ones(1, 1), bias)
    assert module.bias.is_contiguous() and torch.equal(module.bias, bias)


@pytest.mark.parametrize("dtype", [torch.int32, torch.float64, torch.bool])
def test_a_bias_that_no_call_takes_is_refused(dtype):
    with pytest.raises(ValueError, match="bias"):
        FrozenFp8Linear.from_codes(_codes(20, 32), torch.ones(1, 1), torch.zeros(20).to(dtype))
