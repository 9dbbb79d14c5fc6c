"""Coded activations without a GPU: the entry points' argument checks and the loud refusal of CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

from moss_image_b200 import _lib
from moss_image_b200.activation_codes import (CodedActivation, coded_linear, coded_weight_gradient, decode_activation,
                                              encode_activation)


def test_encode_and_decode_validate_arguments():
    lib = _lib.library()

    def encode(x=64, dtype=1, rows=4, cols=64, codes=64, ld=64, exponents=64):
        return lib.moss_codes_encode(x, dtype, rows, cols, codes, ld, exponents, None)

    assert encode(rows=0) == _lib.MOSS_OK and encode(cols=0) == _lib.MOSS_OK
    assert encode(x=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert encode(codes=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert encode(exponents=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert encode(codes=68) == _lib.MOSS_ERR_INVALID_ARGUMENT  # unaligned rows
    assert encode(ld=63) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert encode(ld=80) == _lib.MOSS_ERR_INVALID_ARGUMENT  # not the least pitch
    assert encode(rows=-1) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert encode(rows=1 << 40) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert encode(dtype=5) == _lib.MOSS_ERR_UNSUPPORTED
    assert lib.moss_codes_decode(64, 40, 64, 4, 40, 64, 1, None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert lib.moss_codes_decode(64, 48, 64, 4, 40, None, 1, None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert lib.moss_codes_decode(64, 48, 64, 4, 40, 64, 9, None) == _lib.MOSS_ERR_UNSUPPORTED


def test_gradient_validates_arguments():
    lib = _lib.library()
    size = ctypes.c_size_t()
    assert lib.moss_coded_gradient_workspace_bytes(1000, 64, 640, ctypes.byref(size)) == _lib.MOSS_OK
    assert size.value >= 1000 * (640 + 64) * 2  # decoded rows, and room for a copy of the gradient's
    assert lib.moss_coded_gradient_workspace_bytes(0, 64, 640, ctypes.byref(size)) == _lib.MOSS_OK and size.value == 0
    assert lib.moss_coded_gradient_workspace_bytes(4, -1, 640, ctypes.byref(size)) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert lib.moss_coded_gradient_workspace_bytes(4, 1 << 23, 640, ctypes.byref(size)) == _lib.MOSS_ERR_INVALID_ARGUMENT

    def gradient(dy=64, dtype=1, n=64, codes=64, ld=640, dw=64, out=1, workspace=None, size=0):
        return lib.moss_coded_gradient(dy, dtype, 1000, n, codes, ld, 64, 640, dw, out, workspace, size, None, None)

    assert gradient(n=0) == _lib.MOSS_OK
    assert gradient(dtype=2) == _lib.MOSS_ERR_UNSUPPORTED  # float32 gradients
    assert gradient(out=4) == _lib.MOSS_ERR_UNSUPPORTED
    assert gradient(dy=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert gradient(dw=None) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert gradient(ld=632) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert gradient() == _lib.MOSS_ERR_INVALID_ARGUMENT and "workspace" in _lib.last_error()
    assert gradient(workspace=256, size=1024) == _lib.MOSS_ERR_INVALID_ARGUMENT
    assert gradient(workspace=264, size=1 << 40) == _lib.MOSS_ERR_INVALID_ARGUMENT


def test_cpu_tensors_are_refused():
    x = torch.ones(2, 32, dtype=torch.bfloat16)
    codes, exponents = torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 1, dtype=torch.uint8)
    for call in (lambda: encode_activation(x), lambda: coded_weight_gradient(x, codes, exponents), lambda: coded_linear(x, x),
                 lambda: decode_activation(CodedActivation(codes, exponents, x.shape, x.dtype))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()
