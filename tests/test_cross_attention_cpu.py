"""Attention to another sequence without a GPU: the entry points' argument checks and the loud refusal of CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moss_image_b200 import _lib
from moss_image_b200.cross_attention import cross_attention, cross_attention_packed


def _forward(q=256, dtype=1, batch=2, tq=300, tk=200, hq=4, hk=2, dim=64, offsets=(None, None), mask=None, scale=0.125,
             out=256, workspace=None, size=0):
    rows = (0, hk * dim, dim)
    return _lib.library().moss_cross_attention_fwd(q, 0, hq * dim, dim, 256, *rows, 256, *rows, dtype, batch, tq, tk, hq, hk, dim,
                                                   *offsets, mask, tk, scale, out, None, workspace, size, None, None)


def test_forward_validates_arguments():
    assert _forward(tq=0) == _lib.MOSS_OK
    assert _forward(batch=0) == _lib.MOSS_OK
    assert _forward(dtype=2) == _lib.MOSS_ERR_UNSUPPORTED
    assert _forward(dim=60) == _lib.MOSS_ERR_UNSUPPORTED
    assert _forward(dim=136) == _lib.MOSS_ERR_UNSUPPORTED
    assert _forward(hq=3) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(hk=0) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(tq=-1) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(tq=1 << 40) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(scale=0.0) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(scale=float("nan")) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(offsets=(256, None)) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(offsets=(256, 256), mask=256) == _lib.MOSS_ERR_UNSUPPORTED
    assert _forward(out=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(q=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert _forward(batch=1, tq=1, tk=4096, hq=1, hk=1) == _lib.MOSS_ERR_INVALID_ARGUMENT  # splits without a workspace
    assert "workspace" in _lib.last_error()


def test_workspace_and_backward_validate_arguments():
    lib = _lib.library()
    size = ctypes.c_size_t()

    def room(*sizes, packed=0, backward=0):
        assert lib.moss_cross_attention_workspace_bytes(*sizes, packed, backward, ctypes.byref(size)) == _lib.MOSS_OK
        return size.value

    assert room(2, 4096, 512, 24, 24, 128) == 0  # enough units: no splits
    assert room(1, 1, 4096, 1, 1, 128) > 0
    assert room(2, 4096, 512, 24, 24, 128, backward=1) >= 2 * 4096 * 24 * 4  # a delta for each row and head
    assert room(2, 0, 512, 24, 24, 128, backward=1) == 0
    assert room(5, 4096, 512, 24, 8, 64, packed=1, backward=1) >= 4096 * 24 * 4
    assert lib.moss_cross_attention_workspace_bytes(2, 8, 8, 3, 2, 64, 0, 0, ctypes.byref(size)) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert lib.moss_cross_attention_workspace_bytes(2, 8, 8, 2, 2, 64, 0, 0, None) == _lib.MOSS_ERR_INVALID_ARGUMENT

    def backward(dq=256, dk=256, dv=256, lse=256, workspace=256, size=1 << 40):
        rows = (0, 128, 64)
        return lib.moss_cross_attention_bwd(256, 256, *rows, 256, *rows, 256, *rows, 1, 1, 300, 200, 2, 2, 64, None, None, None,
                                            0, 0.125, 256, lse, dq, dk, dv, workspace, size, None, None)

    assert backward(dk=None) == _lib.MOSS_ERR_INVALID_ARGUMENT  # the two come together
    assert backward(dq=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert backward(lse=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert backward(workspace=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert backward(size=64) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert backward(workspace=272) == _lib.MOSS_ERR_INVALID_ARGUMENT


def test_cpu_tensors_are_refused():
    x = torch.ones(1, 2, 1, 8, dtype=torch.bfloat16)
    offsets = torch.tensor([0, 2])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        cross_attention(x, x, x)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        cross_attention_packed(x[0], x[0], x[0], offsets, offsets)
