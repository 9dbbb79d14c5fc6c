"""Layer norm without a GPU: the entry points' argument checks and the loud refusal of CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moss_image_b200 import _lib
from moss_image_b200.norms import layer_norm


def test_entry_points_validate_arguments():
    lib = _lib.library()

    def forward(rows=4, dim=64, dtype=1, gain=1, weight=None):
        return lib.moss_layernorm_fwd(None, dtype, rows, dim, weight, None, gain, 1e-6, None, None, None)

    assert forward(rows=0) == _lib.MOSS_OK
    assert forward() == _lib.MOSS_ERR_INVALID_ARGUMENT  # null pointers
    assert forward(dim=0) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert forward(rows=-1) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert forward(dtype=7) == _lib.MOSS_ERR_UNSUPPORTED
    assert forward(dim=16385) == _lib.MOSS_ERR_UNSUPPORTED
    assert "16384" in _lib.last_error()
    assert forward(gain=9, weight=64) == _lib.MOSS_ERR_UNSUPPORTED

    size = ctypes.c_size_t()
    assert lib.moss_layernorm_bwd_workspace_bytes(1000, 640, ctypes.byref(size)) == _lib.MOSS_OK
    assert size.value >= 2 * 640 * 4
    assert lib.moss_layernorm_bwd_workspace_bytes(1000, 640, None) == _lib.MOSS_ERR_INVALID_ARGUMENT

    def backward(gain, dw, workspace=None, size=0):
        return lib.moss_layernorm_bwd(256, 256, 1, 4, 64, None, 1, 256, gain, None, dw, None, workspace, size, None)

    assert backward(0, 256) == _lib.MOSS_ERR_INVALID_ARGUMENT  # no gain in the forward pass
    assert backward(1, 256) == _lib.MOSS_ERR_INVALID_ARGUMENT  # no workspace
    assert backward(1, 256, 256, 16) == _lib.MOSS_ERR_INVALID_ARGUMENT  # a small one
    assert backward(1, None) == _lib.MOSS_OK  # nothing is asked for


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        layer_norm(torch.ones(2, 8))
