"""Saved activations as 8-bit codes, and the weight gradients that read them.

What the forward pass keeps for the backward one is half of a step's memory, and
:mod:`moss_image_b200.activation_offload` moves it out whole. Here it is kept in half the bytes: int8
codes with one power of two for each 32 values of a row (:func:`encode_activation`), 8.25 bits a value. A
decoded value is within 1/127 of its block's largest magnitude (or within 2^-127, in blocks below 2^-119) and, since a
code has seven bits and a sign, exact in the activation's own type, so that what a product reads is what the codes stand for.

* :func:`encode_activation` / :func:`decode_activation`: the codes on their own. A block with an infinity
  or NaN decodes to NaN.
* :func:`coded_weight_gradient`: ``dW = dY^T decode(X)`` on the tensor cores, from the codes.
* :func:`coded_linear`: a trainable linear that keeps its input as codes. Several linears of one input
  (q, k and v) share them through ``coded=``.
* :func:`coded_checkpoints`: a scope in which a checkpointed block's input is kept as codes; the
  backward pass recomputes the block from the decoded input.

CUDA tensors only: there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Callable, ContextManager, NamedTuple

import torch
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import _lib
from .quant_kernels import _poll_after_backward, poll_device_status, status_buffer

CODE_BLOCK = 32
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_FEW_FEATURES = 32  # gradients that the kernels read in place whatever their alignment is


class CodedActivation(NamedTuple):
    """``codes``: int8 ``[rows, columns]`` whose rows start 16 bytes apart or a multiple of it; ``exponents``:
    uint8 ``[rows, ceil(columns / 32)]``, a power of two plus 127 each; what they decode to by default."""

    codes: torch.Tensor
    exponents: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype


def _blocks(columns: int) -> int:
    return -(-columns // CODE_BLOCK)


def encode_activation(tokens: torch.Tensor) -> CodedActivation:
    """Codes of ``[..., columns]`` float16, bfloat16 or float32 CUDA tokens (strided ones are copied first)."""
    if not tokens.is_cuda:
        raise RuntimeError("encode_activation runs on CUDA tensors only (there is no CPU path).")
    if tokens.dtype not in _FLOATS or tokens.ndim < 1:
        raise ValueError("encode_activation: tokens must be [..., columns] of float16, bfloat16 or float32.")
    _lib.refuse_forward_mode("encode_activation", tokens)
    device = tokens.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return encode_activation(tokens)
    dense = tokens.detach().contiguous()
    columns = dense.shape[-1]
    rows = math.prod(dense.shape[:-1])
    pitch = -(-columns // 16) * 16
    codes = torch.empty(rows, pitch, dtype=torch.int8, device=device)
    exponents = torch.empty(rows, _blocks(columns), dtype=torch.uint8, device=device)
    _lib.check(_lib.library().moss_codes_encode(
        dense.data_ptr(), _lib.DTYPE_CODES[dense.dtype], rows, columns, codes.data_ptr(), pitch, exponents.data_ptr(),
        _lib.stream_handle(device)), "moss_codes_encode")
    _lib.count_launch("codes")
    return CodedActivation(codes if pitch == columns else codes[:, :columns], exponents, tokens.shape, tokens.dtype)


def _check_codes(codes: torch.Tensor, exponents: torch.Tensor, what: str) -> torch.Tensor:
    """The codes, with rows as the kernels read them."""
    if not codes.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA tensors only (there is no CPU path).")
    if codes.dtype != torch.int8 or codes.ndim != 2 or exponents.dtype != torch.uint8:
        raise ValueError(f"{what}: codes must be int8 [rows, columns] with uint8 exponents.")
    rows, columns = codes.shape
    if exponents.device != codes.device or exponents.shape != (rows, _blocks(columns)) or not exponents.is_contiguous():
        raise ValueError(f"{what}: exponents must be a contiguous [rows, ceil(columns / 32)] tensor on the codes' device.")
    pitch, step = codes.stride()
    if rows and columns and (step != 1 or pitch % 16 or pitch < columns or codes.data_ptr() % 16
                             or _room(codes) < rows * pitch):
        held = torch.zeros(rows, -(-columns // 16) * 16, dtype=torch.int8, device=codes.device)
        held[:, :columns] = codes
        codes = held[:, :columns]
    return codes


def _room(codes: torch.Tensor) -> int:
    """Bytes from the first code to the end of its storage: rows are read whole, up to a multiple of 16."""
    return codes.untyped_storage().nbytes() - codes.storage_offset()


def _pitch(codes: torch.Tensor) -> int:
    return codes.stride(0) if codes.numel() else -(-codes.shape[1] // 16) * 16


def decode_activation(coded: CodedActivation, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values that the codes stand for, in the shape that was encoded; ``dtype`` defaults to what it had."""
    codes = _check_codes(coded.codes, coded.exponents, "decode_activation")
    dtype = coded.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise ValueError("decode_activation: the output must be float16, bfloat16 or float32.")
    if len(coded.shape) < 1 or math.prod(coded.shape[:-1]) != codes.shape[0] or coded.shape[-1] != codes.shape[1]:
        raise ValueError("decode_activation: the codes do not have the shape that was encoded.")
    device = codes.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return decode_activation(coded, dtype)
    out = torch.empty(coded.shape, dtype=dtype, device=device)
    _lib.check(_lib.library().moss_codes_decode(
        codes.data_ptr(), _pitch(codes), coded.exponents.data_ptr(), codes.shape[0], codes.shape[1], out.data_ptr(),
        _lib.DTYPE_CODES[dtype], _lib.stream_handle(device)), "moss_codes_decode")
    _lib.count_launch("codes")
    return out


def _holds(dtype: torch.dtype, coded_dtype: torch.dtype) -> bool:
    """Whether products in ``dtype`` can read codes of ``coded_dtype`` tokens as what they stand for."""
    return dtype != torch.float16 or coded_dtype == torch.float16


@lru_cache(maxsize=1024)
def _workspace_bytes(device: int, rows: int, features: int, columns: int) -> int:
    size = ctypes.c_size_t()
    with torch.cuda.device(device):  # the plan counts its multiprocessors
        _lib.check(_lib.library().moss_coded_gradient_workspace_bytes(rows, features, columns, ctypes.byref(size)),
                   "moss_coded_gradient_workspace_bytes")
    return size.value


class _WithoutGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gradient, codes, exponents, output_dtype, coded_dtype):
        return coded_weight_gradient(gradient, codes, exponents, output_dtype, coded_dtype=coded_dtype)

    @staticmethod
    def backward(ctx, gradient):
        raise NotImplementedError("coded_weight_gradient has no gradient (no second derivatives).")


def coded_weight_gradient(gradient: torch.Tensor, codes: torch.Tensor, exponents: torch.Tensor,
                          output_dtype: torch.dtype | None = None, *,
                          coded_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``dW = dY^T decode(X)``: ``[features, columns]`` from ``[..., features]`` float16 or bfloat16 gradients and the
    codes of the ``[..., columns]`` input. Sums are float32, in a fixed order, rounded once to ``output_dtype``
    (the gradient's own by default).

    ``coded_dtype``: what the codes were made from, the gradient's dtype where it is not given. The product reads decoded
    values in the gradient's dtype: bfloat16 holds those of any codes, float16 those of float16 tokens only. Not
    differentiable: a backward pass that reaches a result whose gradient input requires grad raises.
    """
    what = "coded_weight_gradient"
    if not gradient.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA tensors only (there is no CPU path).")
    if gradient.dtype not in (torch.float16, torch.bfloat16) or gradient.ndim < 1:
        raise ValueError(f"{what}: the gradient must be [..., features] of float16 or bfloat16.")
    if codes.device != gradient.device:
        raise ValueError(f"{what}: codes must be on the gradient's device.")
    dtype = gradient.dtype if output_dtype is None else output_dtype
    if dtype not in _FLOATS:
        raise ValueError(f"{what}: the output must be float16, bfloat16 or float32.")
    if not _holds(gradient.dtype, gradient.dtype if coded_dtype is None else coded_dtype):
        raise ValueError(f"{what}: float16 does not hold what codes of {coded_dtype} tokens stand for.")
    _lib.refuse_forward_mode(what, gradient)
    if torch.is_grad_enabled() and gradient.requires_grad:
        return _WithoutGradient.apply(gradient, codes, exponents, output_dtype, coded_dtype)
    device = gradient.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return coded_weight_gradient(gradient, codes, exponents, output_dtype, coded_dtype=coded_dtype)
    codes = _check_codes(codes, exponents, what)
    rows, columns = codes.shape
    features = gradient.shape[-1]
    if math.prod(gradient.shape[:-1]) != rows:
        raise ValueError(f"{what}: the gradient must have one row for each row of codes.")
    status = status_buffer(device)
    poll_device_status(device)
    gradient = gradient.detach().contiguous()
    out = torch.empty(features, columns, dtype=dtype, device=device)
    size = _workspace_bytes(device.index, rows, features, columns)
    if size and features > _FEW_FEATURES and features % 8 == 0 and gradient.data_ptr() % 16 == 0:
        size -= -(-rows * features * 2 // 256) * 256  # read in place: no room for a copy
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.check(_lib.library().moss_coded_gradient(
        gradient.data_ptr(), _lib.DTYPE_CODES[gradient.dtype], rows, features, codes.data_ptr(), _pitch(codes),
        exponents.data_ptr(), columns, out.data_ptr(), _lib.DTYPE_CODES[dtype], _lib.ptr(workspace), size,
        status.data_ptr(), _lib.stream_handle(device)), "moss_coded_gradient")
    _lib.count_launch("codes")
    return out


class _CodedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, bias, codes, exponents):
        ctx.save_for_backward(weight, codes, exponents)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return F.linear(tokens, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, gradient):
        weight, codes, exponents = ctx.saved_tensors
        _lib.refuse_forward_mode("coded_linear", gradient)
        d_tokens = d_weight = d_bias = None
        if ctx.needs_input_grad[0]:
            d_tokens = gradient @ weight
        if ctx.needs_input_grad[1]:
            _poll_after_backward(gradient.device)
            d_weight = coded_weight_gradient(gradient, codes, exponents, weight.dtype)
        if ctx.needs_input_grad[2]:
            rows = math.prod(gradient.shape[:-1])  # (a row of no features tells no number of rows)
            d_bias = gradient.reshape(rows, gradient.shape[-1]).sum(0, dtype=torch.float32).to(ctx.bias_dtype)
        return d_tokens, d_weight, d_bias, None, None


def codes_serve(tokens: torch.Tensor, weight_dtype: torch.dtype) -> bool:
    """Whether :func:`coded_linear` takes the tokens with a weight of this dtype, under the autocast that is on."""
    if not tokens.is_cuda or tokens.dtype not in (torch.float16, torch.bfloat16) or weight_dtype != tokens.dtype:
        return False
    return not torch.is_autocast_enabled("cuda") or torch.get_autocast_dtype("cuda") == tokens.dtype


def coded_linear(tokens: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                 coded: CodedActivation | None = None) -> torch.Tensor:
    """``F.linear(tokens, weight, bias)`` that keeps its input as codes for the weight's gradient.

    float16 or bfloat16, one dtype. The output and the input's gradient are those of ``F.linear``; only the weight's
    gradient sees the codes. ``coded``: the codes of these tokens (:func:`encode_activation`), made here where they are not given.
    """
    if not tokens.is_cuda:
        raise RuntimeError("coded_linear runs on CUDA tensors only (there is no CPU path).")
    given = [tokens, weight] if bias is None else [tokens, weight, bias]
    if tokens.dtype not in (torch.float16, torch.bfloat16) or any(t.dtype != tokens.dtype for t in given):
        raise ValueError("coded_linear: tokens, weight and bias must have one dtype of float16 or bfloat16.")
    if any(t.device != tokens.device for t in given):
        raise ValueError("coded_linear: tokens, weight and bias must be on one device.")
    if tokens.ndim < 1 or weight.ndim != 2 or weight.shape[1] != tokens.shape[-1]:
        raise ValueError("coded_linear: the weight must be [out, in] for [..., in] tokens.")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError("coded_linear: the bias must be [out].")
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") != tokens.dtype:
        raise ValueError("coded_linear: autocast runs in another dtype than the tokens and the weight have.")
    if coded is not None and (coded.shape != tokens.shape or coded.codes.device != tokens.device):
        raise ValueError("coded_linear: the codes are not those of these tokens (another shape or device).")
    if coded is not None and coded.dtype != tokens.dtype:
        raise ValueError("coded_linear: the codes are those of tokens of another dtype.")
    _lib.refuse_forward_mode("coded_linear", *given)
    if not torch.is_grad_enabled() or not any(t.requires_grad for t in given):
        return F.linear(tokens, weight, bias)
    if not weight.requires_grad:  # nothing of the input is kept
        return F.linear(tokens, weight, bias)
    if coded is None:
        coded = encode_activation(tokens)
    return _CodedLinear.apply(tokens, weight, bias, coded.codes, coded.exponents)


def coded_checkpoints(tokens: torch.Tensor, outer: ContextManager | None = None) -> ContextManager:
    """A scope for one ``checkpoint`` call (non-reentrant) of a block on ``tokens``: what it keeps of the tokens are codes.

    The tokens are coded where autograd saves them in the scope; everything else that it saves is kept as it is, other
    tensors of their shape too. ``outer``: the saved-tensor hooks of the scope around it (``activation_cpu_offload``), which then
    receive the codes and everything else.
    """
    def same(value: torch.Tensor) -> torch.Tensor:
        return value

    hide: Callable = getattr(outer, "pack_hook", same)
    show: Callable = getattr(outer, "unpack_hook", same)
    codable = tokens.is_cuda and tokens.dtype in _FLOATS and tokens.ndim >= 1
    # (the caller holds the tokens while the scope is open: nothing else has their address)
    which = (tokens.data_ptr(), tokens.shape, tokens.stride(), tokens.dtype)

    def pack(saved: torch.Tensor):
        if not codable or not saved.is_cuda or (saved.data_ptr(), saved.shape, saved.stride(), saved.dtype) != which:
            return hide(saved), None, None
        codes, exponents, *meant = encode_activation(saved)
        return hide(codes), hide(exponents), meant

    def unpack(packed):
        held, exponents, meant = packed
        if meant is None:
            return show(held)
        return decode_activation(CodedActivation(show(held), show(exponents), *meant))

    return torch.autograd.graph.saved_tensors_hooks(pack, unpack)
