"""Frozen linears in block-scaled 8-bit floating point, executed by the sm_100a kernels.

The sibling of the int8 linear (:mod:`moss_image_b200.quantization`) for weights held as e4m3
codes with one float32 scale per 128 x 128 block. There the weight is decoded to 16 bits on its
way to the tensor cores; here activations and gradients are quantised too, per row and 128
columns inside the call, and the products run on the 8-bit tensor-core path at twice the rate.
Forward and input gradient read the same ``[out, in]`` codes; no decoded or transposed copy of
the weight exists. Gradients flow to the input only (training/quantization.py:27-65).

A row's scale is the least power of two that brings the block within the format's +-448, so a
code does not depend on how a division rounds. Sums are held in float32 and rounded once, to the
output type. Codes have 4 significant bits: expect about 3 percent of noise (relative 2-norm) on
each quantised operand, averaged down by the sums. An infinity or NaN in a row gives a NaN row.

CUDA tensors only: there is no CPU path and no fallback.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .quant_kernels import _poll_after_backward, autocast_compute_dtype, poll_device_status, status_buffer
from .quantization import replace_frozen_linears

BLOCK = 128
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def _blocks(size: int) -> int:
    return -(-size // BLOCK)


def _pitched_codes(rows: int, columns: int, device: torch.device) -> torch.Tensor:
    """Zeroed e4m3 ``[rows, columns]`` whose rows start 16 bytes apart or a multiple of it (the TMA's rule)."""
    pitch = -(-columns // 16) * 16
    return torch.zeros(rows, pitch, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)[:, :columns]


def lay_out_fp8_codes(codes: torch.Tensor) -> torch.Tensor:
    """The codes as the kernels read them: as they are when their rows are 16-byte aligned, else a
    copy with padded rows (an input width that is no multiple of 16)."""
    if codes.dtype != torch.float8_e4m3fn or codes.ndim != 2:
        raise ValueError("fp8 codes must be a float8_e4m3fn [out, in] tensor.")
    if codes.stride(1) == 1 and codes.stride(0) % 16 == 0 and codes.stride(0) >= codes.shape[1] and codes.data_ptr() % 16 == 0:
        return codes
    held = _pitched_codes(codes.shape[0], codes.shape[1], codes.device)
    held.view(torch.uint8).copy_(codes.view(torch.uint8))
    return held


def _padded_codes(codes: torch.Tensor) -> torch.Tensor:
    """The codes as whole padded rows, ``[out, ceil(in / 16) * 16]`` without gaps, so that any dense copy of them keeps the
    kernels' row pitch. The same memory where it is laid out like that already."""
    codes = lay_out_fp8_codes(codes)
    rows, columns = codes.shape
    pitch = -(-columns // 16) * 16
    if rows == 0 or columns == 0:
        return codes.new_empty(rows, pitch)
    room = codes.untyped_storage().nbytes() - codes.storage_offset()
    if codes.stride(0) == pitch and room >= rows * pitch:
        return codes.as_strided((rows, pitch), (pitch, 1))
    held = _pitched_codes(rows, pitch, codes.device)
    held[:, :columns].view(torch.uint8).copy_(codes.view(torch.uint8))
    return held


def quantize_fp8_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes ``[out, in]`` and float32 scales ``[ceil(out / 128), ceil(in / 128)]`` of a CUDA weight.

    A block's scale is ``max|w| / 448``. Raises ``ValueError`` on non-finite weights.
    """
    if weight.ndim != 2 or weight.dtype not in _FLOATS:
        raise ValueError("fp8 weights are quantized from a float [out, in] matrix.")
    if not weight.is_cuda:
        raise RuntimeError("fp8 linears run on CUDA tensors only (there is no CPU path).")
    if weight.get_device() != _lib.current_device_index():
        with torch.cuda.device(weight.device):
            return quantize_fp8_weight(weight)
    weight = weight.contiguous()
    rows, columns = weight.shape
    codes = _pitched_codes(rows, columns, weight.device)
    scale = torch.zeros(_blocks(rows), _blocks(columns), device=weight.device)
    status = torch.zeros(1, dtype=torch.int32, device=weight.device)
    _lib.check(_lib.library().moss_fp8_quantize_weight(
        weight.data_ptr(), _lib.dtype_code(weight.dtype), rows, columns, codes.data_ptr(), -(-columns // 16) * 16,
        scale.data_ptr(), status.data_ptr(), _lib.stream_handle(weight.device)), "moss_fp8_quantize_weight")
    _lib.count_launch("fp8_quantize")
    if int(status.item()) & _lib.STATUS_NONFINITE_WEIGHT:
        raise ValueError("Cannot quantize non-finite weights.")
    return codes, scale


def quantize_fp8_rows(tokens: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The row quantiser of the linear on its own: codes ``[rows, k]`` and float32 scales
    ``[rows, ceil(k / 128)]`` of a CUDA matrix. The scales are powers of two."""
    if tokens.ndim != 2 or tokens.dtype not in _FLOATS:
        raise ValueError("fp8 rows are quantized from a float [rows, k] matrix.")
    if not tokens.is_cuda:
        raise RuntimeError("fp8 linears run on CUDA tensors only (there is no CPU path).")
    if tokens.get_device() != _lib.current_device_index():
        with torch.cuda.device(tokens.device):
            return quantize_fp8_rows(tokens)
    tokens = tokens.contiguous()
    rows, columns = tokens.shape
    codes = torch.empty(rows, _blocks(columns) * BLOCK, dtype=torch.uint8, device=tokens.device)
    scale = torch.empty(_blocks(columns), rows, device=tokens.device)
    _lib.check(_lib.library().moss_fp8_quantize_rows(
        tokens.data_ptr(), _lib.dtype_code(tokens.dtype), rows, columns, codes.data_ptr(), scale.data_ptr(), rows,
        _lib.stream_handle(tokens.device)), "moss_fp8_quantize_rows")
    _lib.count_launch("fp8_quantize")
    return codes.view(torch.float8_e4m3fn)[:, :columns], scale.t()


@lru_cache(maxsize=1024)
def _workspace_bytes(device: int, m: int, n_out: int, k_red: int) -> int:
    size = ctypes.c_size_t()
    with torch.cuda.device(device):  # the plan counts its multiprocessors
        _lib.check(_lib.library().moss_fp8_linear_workspace_bytes(m, n_out, k_red, ctypes.byref(size)),
                   "moss_fp8_linear_workspace_bytes")
    return size.value


def _check(tokens: torch.Tensor, weight: torch.Tensor, k: int, scale: torch.Tensor, side: int, what: str) -> None:
    """``k``: columns of the weight, whose rows may be padded; ``side``: its dimension that the input's last one has to match."""
    if not tokens.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA tensors only (there is no CPU path).")
    if tokens.dtype not in _FLOATS:
        raise ValueError(f"{what}: the input must be float16, bfloat16 or float32.")
    device = tokens.get_device()
    if weight.get_device() != device or scale.get_device() != device:
        raise ValueError(f"{what}: the weight and its scales must be on the input's device.")
    if weight.dtype != torch.float8_e4m3fn or weight.ndim != 2 or scale.dtype != torch.float32:
        raise ValueError(f"{what}: the weight must be float8_e4m3fn [out, in] with float32 scales.")
    n = weight.shape[0]
    if scale.shape != (-(-n // BLOCK), -(-k // BLOCK)) or not scale.is_contiguous():
        raise ValueError(f"{what}: the scales must be a contiguous [ceil(out / 128), ceil(in / 128)] tensor.")
    if tokens.ndim < 1 or tokens.shape[-1] != (k if side else n):
        raise ValueError(f"{what}: the input's last dimension must be {k if side else n}.")
    pitch, step = weight.stride()
    if n and k and (step != 1 or pitch % 16 or pitch < k or weight.data_ptr() % 16):
        raise ValueError(f"{what}: the weight's rows must be 16-byte aligned (lay_out_fp8_codes).")


def _output(tokens: torch.Tensor, width: int, dtype: torch.dtype, out: torch.Tensor | None, what: str) -> torch.Tensor:
    shape = (*tokens.shape[:-1], width)
    if dtype not in _FLOATS:
        raise ValueError(f"{what}: the output must be float16, bfloat16 or float32.")
    if out is None:
        return tokens.new_empty(shape) if dtype is tokens.dtype else tokens.new_empty(shape, dtype=dtype)
    if tuple(out.shape) != shape or out.dtype != dtype or out.device != tokens.device or not out.is_contiguous():
        raise ValueError(f"{what}: the output buffer has the wrong shape, dtype or device or is not contiguous.")
    return out


def _rows(tokens: torch.Tensor) -> int:
    return tokens.shape[0] if tokens.ndim == 2 else math.prod(tokens.shape[:-1])


def fp8_linear_forward(tokens: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor,
                       bias: torch.Tensor | None = None, output_dtype: torch.dtype | None = None, *,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """``Y = q(X) dec(W)^T (+ bias)`` for ``[..., in]`` tokens; ``output_dtype`` defaults to the tokens' own."""
    return _forward(tokens, weight, None, scale, bias, output_dtype, out)


def _forward(tokens: torch.Tensor, weight: torch.Tensor, columns: int | None, scale: torch.Tensor, bias: torch.Tensor | None,
             output_dtype: torch.dtype | None, out: torch.Tensor | None) -> torch.Tensor:
    what = "fp8_linear_forward"
    n, k = weight.shape if weight.ndim == 2 else (0, 0)
    k = k if columns is None else columns
    _check(tokens, weight, k, scale, 1, what)
    if tokens.get_device() != _lib.current_device_index():
        with torch.cuda.device(tokens.device):
            return _forward(tokens, weight, columns, scale, bias, output_dtype, out)
    if bias is not None and (bias.device != tokens.device or tuple(bias.shape) != (n,) or bias.dtype not in _FLOATS
                             or not bias.is_contiguous()):
        raise ValueError(f"{what}: the bias must be a contiguous float [out] tensor on the input's device.")
    device = tokens.device
    status = status_buffer(device)
    poll_device_status(device)
    tokens = tokens.contiguous()
    output = _output(tokens, n, output_dtype or tokens.dtype, out, what)
    rows = _rows(tokens)
    size = _workspace_bytes(device.index, rows, n, k)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.check(_lib.library().moss_fp8_linear_fwd(
        tokens.data_ptr(), _lib.DTYPE_CODES[tokens.dtype], rows, k, weight.data_ptr(), weight.stride(0),
        scale.data_ptr(), n, _lib.ptr(bias), 0 if bias is None else _lib.DTYPE_CODES[bias.dtype], output.data_ptr(),
        _lib.DTYPE_CODES[output.dtype], _lib.ptr(workspace), size, status.data_ptr(), _lib.stream_handle(device)),
        "moss_fp8_linear_fwd")
    _lib.count_launch("fp8_linear")
    return output


def fp8_linear_backward(gradient: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor,
                        output_dtype: torch.dtype | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """``dX = q(dY) dec(W)`` for ``[..., out]`` gradients, from the same ``[out, in]`` codes."""
    return _backward(gradient, weight, None, scale, output_dtype, out)


def _backward(gradient: torch.Tensor, weight: torch.Tensor, columns: int | None, scale: torch.Tensor,
              output_dtype: torch.dtype | None, out: torch.Tensor | None) -> torch.Tensor:
    what = "fp8_linear_backward"
    n, k = weight.shape if weight.ndim == 2 else (0, 0)
    k = k if columns is None else columns
    _check(gradient, weight, k, scale, 0, what)
    if gradient.get_device() != _lib.current_device_index():
        with torch.cuda.device(gradient.device):
            return _backward(gradient, weight, columns, scale, output_dtype, out)
    device = gradient.device
    status = status_buffer(device)
    poll_device_status(device)
    gradient = gradient.contiguous()
    output = _output(gradient, k, output_dtype or gradient.dtype, out, what)
    rows = _rows(gradient)
    size = _workspace_bytes(device.index, rows, k, n)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.check(_lib.library().moss_fp8_linear_dx(
        gradient.data_ptr(), _lib.DTYPE_CODES[gradient.dtype], rows, n, weight.data_ptr(), weight.stride(0),
        scale.data_ptr(), k, output.data_ptr(), _lib.DTYPE_CODES[output.dtype], _lib.ptr(workspace), size,
        status.data_ptr(), _lib.stream_handle(device)), "moss_fp8_linear_dx")
    _lib.count_launch("fp8_linear")
    return output


class _Fp8Linear(torch.autograd.Function):
    """Saves only the weight's codes and scales, as the int8 linear does (training/quantization.py:29-45)."""

    @staticmethod
    def forward(ctx, tokens, weight, columns, scale, bias, output_dtype):
        ctx.save_for_backward(weight, scale)
        ctx.input_dtype, ctx.columns = tokens.dtype, columns
        return _forward(tokens, weight, columns, scale, bias, output_dtype, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, gradient):
        weight, scale = ctx.saved_tensors
        _lib.refuse_forward_mode("fp8_linear", gradient)
        _poll_after_backward(gradient.device)
        return _backward(gradient, weight, ctx.columns, scale, ctx.input_dtype, None), None, None, None, None, None


def fp8_linear(tokens: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None,
               output_dtype: torch.dtype | None = None) -> torch.Tensor:
    """:func:`fp8_linear_forward`, differentiable in ``tokens`` (weight, scales and bias are frozen)."""
    return _linear(tokens, weight, None, scale, bias, output_dtype)


def _linear(tokens: torch.Tensor, weight: torch.Tensor, columns: int | None, scale: torch.Tensor, bias: torch.Tensor | None,
            output_dtype: torch.dtype | None) -> torch.Tensor:
    _lib.refuse_forward_mode("fp8_linear", tokens)
    if torch.is_grad_enabled() and tokens.requires_grad:
        return _Fp8Linear.apply(tokens, weight, columns, scale, bias, output_dtype)
    return _forward(tokens, weight, columns, scale, bias, output_dtype, None)


class FrozenFp8Linear(nn.Module):
    """Block-scaled fp8 linear with gradients only to its input.

    Same life as :class:`~moss_image_b200.quantization.FrozenInt8Linear`: built from a frozen
    ``nn.Linear`` on CUDA or from stored codes, usable as the base of a ``LoRALinear``. State:
    ``weight_fp8`` (e4m3 ``[out, in]``), ``weight_scale`` (float32 per block) and ``bias``. The module
    holds the codes with rows padded to 16 bytes (the buffer ``padded_codes``), so that copies of its
    buffers, as block swapping makes them, are laid out as the kernels read them.
    """

    fuses_lora = False  # the adapter's update has its own product

    def __init__(self, linear: nn.Linear) -> None:
        super().__init__()
        if linear.weight.requires_grad or (linear.bias is not None and linear.bias.requires_grad):
            raise ValueError("Freeze the base linear before quantizing it.")
        if linear.weight.device.type == "meta":
            raise ValueError("Load the base weights before quantizing them.")
        codes, scale = quantize_fp8_weight(linear.weight.detach())
        bias = None if linear.bias is None else linear.bias.detach().clone()
        self._set_codes(codes, scale, bias, linear.weight.dtype)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None, *,
                   dtype: torch.dtype = torch.bfloat16) -> "FrozenFp8Linear":
        """Wrap a checkpoint's e4m3 codes ``[out, in]`` and block scales as they are; ``dtype`` is the output's."""
        codes = lay_out_fp8_codes(codes)
        if scale.dtype != torch.float32 or tuple(scale.shape) != (_blocks(codes.shape[0]), _blocks(codes.shape[1])):
            raise ValueError("fp8 scales must be float32 [ceil(out / 128), ceil(in / 128)].")
        if scale.device != codes.device or (bias is not None and bias.device != codes.device):
            raise ValueError("codes, scales and bias must be on one device.")
        if bias is not None and (tuple(bias.shape) != (codes.shape[0],) or bias.dtype not in _FLOATS):
            raise ValueError("bias must be [out], of float16, bfloat16 or float32.")
        module = cls.__new__(cls)
        nn.Module.__init__(module)
        module._set_codes(codes, scale.contiguous(), None if bias is None else bias.contiguous(), dtype)
        return module

    def _set_codes(self, codes: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None, dtype: torch.dtype) -> None:
        self.out_features, self.in_features = codes.shape
        self.register_buffer("padded_codes", _padded_codes(codes), persistent=False)  # saved as weight_fp8
        self.register_buffer("weight_scale", scale)
        self.register_buffer("_dtype_anchor", torch.empty(0, device=codes.device, dtype=dtype), persistent=False)
        self.register_buffer("bias", bias)

    @property
    def compute_dtype(self) -> torch.dtype:
        return self._dtype_anchor.dtype

    @property
    def weight_fp8(self) -> torch.Tensor:
        """The codes ``[out, in]``: a view of the padded rows."""
        codes = self.padded_codes
        return codes if codes.shape[1] == self.in_features else codes[:, :self.in_features]

    @property
    def weight(self) -> torch.Tensor:
        """A transient decoded copy, for inspection (the module itself never makes one)."""
        spread = self.weight_scale.repeat_interleave(BLOCK, 0)[: self.out_features]
        spread = spread.repeat_interleave(BLOCK, 1)[:, : self.in_features]
        return (self.weight_fp8.float() * spread).to(self.compute_dtype)

    def _apply(self, fn, recurse=True):
        # Codes keep their type and scales stay float32 when model.to(dtype=...) casts.
        codes, scale = self.padded_codes, self.weight_scale
        self.padded_codes = codes.view(torch.uint8)
        try:
            result = super()._apply(fn, recurse=recurse)
        finally:
            self.padded_codes = self.padded_codes.view(torch.float8_e4m3fn)
        self.weight_scale = scale.to(device=self._dtype_anchor.device, dtype=torch.float32)
        return result

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        destination[prefix + "weight_fp8"] = self.weight_fp8 if keep_vars else self.weight_fp8.detach()
        super()._save_to_state_dict(destination, prefix, keep_vars)

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        key = prefix + "weight_fp8"
        if key in unexpected_keys:  # it is no buffer of that name
            unexpected_keys.remove(key)
        codes = state_dict.get(key)
        if codes is None:
            if strict:
                missing_keys.append(key)
        elif tuple(codes.shape) != (self.out_features, self.in_features):
            error_msgs.append(f"size mismatch for {key}: {tuple(codes.shape)} in the checkpoint, "
                              f"{(self.out_features, self.in_features)} in the module.")
        elif local_metadata.get("assign_to_params_buffers", False):
            self.padded_codes = _padded_codes(codes.to(torch.float8_e4m3fn))
        else:
            self.weight_fp8.view(torch.uint8).copy_(codes.to(torch.float8_e4m3fn).view(torch.uint8))

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return _linear(tokens, self.padded_codes, self.in_features, self.weight_scale, self.bias,
                       autocast_compute_dtype(tokens, self.compute_dtype))

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def quantize_frozen_linears_fp8(model: nn.Module) -> list[str]:
    """Replace every frozen ``nn.Linear`` below ``model`` (LoRA bases included) by a :class:`FrozenFp8Linear`;
    trainable linears are left alone. Returns the replaced module paths."""
    return replace_frozen_linears(model, FrozenFp8Linear)
