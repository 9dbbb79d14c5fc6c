"""RMSNorm and layer norm of a DiT block on the native kernels (``moss_rmsnorm_*``, ``moss_layernorm_*``).

:func:`rms_norm`: same arithmetic as the reference module (training/model.py:154-172): statistics in f32,
``n = (x * rsqrt(mean(x^2) + eps)).to(x.dtype)``, then ``n * weight`` in torch's promoted
dtype. The kernels keep a row in registers between the two passes and pack several short
rows (the per-head q/k norms) into one warp, so both directions run near the copy bandwidth;
the backward reuses the per-row rsqrt saved by the forward. The sum of squares is reduced in a
different order than torch's, so outputs may differ from the eager module by one rounding of
the result dtype.

:func:`layer_norm`: centred, with an optional gain and offset, both trainable; its backward pass
gives all three gradients in one pass over the rows, summed in a fixed order.

CUDA tensors only: there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from . import _lib


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, eps):
        rows = tokens.reshape(-1, tokens.shape[-1])
        out_dtype = torch.promote_types(tokens.dtype, weight.dtype)
        out = torch.empty(rows.shape, dtype=out_dtype, device=tokens.device)
        rstd = torch.empty(rows.shape[0], dtype=torch.float32, device=tokens.device)
        _lib.check(_lib.library().moss_rmsnorm_fwd(
            rows.data_ptr(), _lib.dtype_code(rows.dtype), rows.shape[0], rows.shape[1], weight.data_ptr(),
            _lib.dtype_code(weight.dtype), float(eps), out.data_ptr(), rstd.data_ptr(),
            _lib.stream_handle(tokens.device)), "moss_rmsnorm_fwd")
        _lib.count_launch("rmsnorm")
        ctx.save_for_backward(rows, weight, rstd)
        ctx.shape = tokens.shape
        return out.view(ctx.shape)

    @staticmethod
    def backward(ctx, grad):
        rows, weight, rstd = ctx.saved_tensors
        out_dtype = torch.promote_types(rows.dtype, weight.dtype)
        grad = grad.reshape(rows.shape).to(out_dtype).contiguous()
        d_tokens = None
        if ctx.needs_input_grad[0]:
            d_rows = torch.empty_like(rows)
            _lib.check(_lib.library().moss_rmsnorm_bwd(
                grad.data_ptr(), rows.data_ptr(), _lib.dtype_code(rows.dtype), rows.shape[0], rows.shape[1],
                weight.data_ptr(), _lib.dtype_code(weight.dtype), rstd.data_ptr(), d_rows.data_ptr(),
                _lib.stream_handle(rows.device)), "moss_rmsnorm_bwd")
            _lib.count_launch("rmsnorm")
            d_tokens = d_rows.view(ctx.shape)
        d_weight = None
        if ctx.needs_input_grad[1]:  # a trainable gain (not on the frozen-base path): torch ops
            normalized = (rows.float() * rstd[:, None]).to(rows.dtype)
            d_weight = (grad.float() * normalized.float()).sum(0).to(weight.dtype)
        return d_tokens, d_weight, None


def rms_norm(tokens: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``(x * rsqrt(mean(x^2) + eps)).to(x.dtype) * weight`` over the last dimension."""
    if not tokens.is_cuda:
        raise RuntimeError("rms_norm runs on CUDA tensors only (there is no CPU path).")
    if weight.shape != tokens.shape[-1:] or weight.device != tokens.device:
        raise ValueError("rms_norm: weight must be [dim] on the tokens' device.")
    return _RMSNorm.apply(tokens.contiguous(), weight.contiguous(), eps)


LAYER_NORM_MAX_DIM = 16384
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


@lru_cache(maxsize=1024)
def _layer_norm_workspace(device: int, rows: int, dim: int) -> int:
    size = ctypes.c_size_t()
    with torch.cuda.device(device):  # the plan counts its multiprocessors
        _lib.check(_lib.library().moss_layernorm_bwd_workspace_bytes(rows, dim, ctypes.byref(size)),
                   "moss_layernorm_bwd_workspace_bytes")
    return size.value


def _gain_code(weight: torch.Tensor | None, bias: torch.Tensor | None) -> int:
    gain = weight if weight is not None else bias
    return 0 if gain is None else _lib.DTYPE_CODES[gain.dtype]


def _layer_norm_forward(tokens, weight, bias, eps, keep_stats):
    device = tokens.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return _layer_norm_forward(tokens, weight, bias, eps, keep_stats)
    gain = weight if weight is not None else bias
    out_dtype = tokens.dtype if gain is None else torch.promote_types(tokens.dtype, gain.dtype)
    out = tokens.new_empty(tokens.shape, dtype=out_dtype)
    dim = tokens.shape[-1]
    rows = math.prod(tokens.shape[:-1])
    stats = torch.empty(rows, 2, dtype=torch.float32, device=device) if keep_stats else None
    _lib.check(_lib.library().moss_layernorm_fwd(
        tokens.data_ptr(), _lib.DTYPE_CODES[tokens.dtype], rows, dim, _lib.ptr(weight), _lib.ptr(bias),
        _gain_code(weight, bias), eps, out.data_ptr(), _lib.ptr(stats), _lib.stream_handle(device)),
        "moss_layernorm_fwd")
    _lib.count_launch("layernorm")
    return out, stats


def _layer_norm_backward(grad, tokens, weight, bias, stats, wanted):
    device = tokens.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return _layer_norm_backward(grad, tokens, weight, bias, stats, wanted)
    dim, rows = tokens.shape[-1], stats.shape[0]
    grad = grad.contiguous()
    d_tokens = torch.empty_like(tokens) if wanted[0] else None
    d_weight = torch.empty_like(weight) if wanted[1] else None
    d_bias = torch.empty_like(bias) if wanted[2] else None
    size = _layer_norm_workspace(device.index, rows, dim) if wanted[1] or wanted[2] else 0
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.check(_lib.library().moss_layernorm_bwd(
        grad.data_ptr(), tokens.data_ptr(), _lib.DTYPE_CODES[tokens.dtype], rows, dim, _lib.ptr(weight),
        _gain_code(weight, bias), stats.data_ptr(), int(weight is not None or bias is not None), _lib.ptr(d_tokens),
        _lib.ptr(d_weight), _lib.ptr(d_bias), _lib.ptr(workspace), size, _lib.stream_handle(device)),
        "moss_layernorm_bwd")
    _lib.count_launch("layernorm")
    return d_tokens, d_weight, d_bias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, bias, eps):
        out, stats = _layer_norm_forward(tokens, weight, bias, eps, True)
        # the offset itself takes no part in the gradients: its type is asked for, not its values
        ctx.save_for_backward(tokens, weight, bias, stats)
        return out

    @staticmethod
    def backward(ctx, grad):
        # (the guard against second derivatives costs microseconds, and is needed where a graph is recorded)
        return _layer_norm_gradients_once(ctx, grad) if torch.is_grad_enabled() else _layer_norm_gradients(ctx, grad)


def _layer_norm_gradients(ctx, grad):
    tokens, weight, bias, stats = ctx.saved_tensors
    _lib.refuse_forward_mode("layer_norm", grad)
    return (*_layer_norm_backward(grad, tokens, weight, bias, stats, ctx.needs_input_grad), None)


_layer_norm_gradients_once = once_differentiable(_layer_norm_gradients)


def layer_norm(tokens: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-6) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, differentiable in all three.

    ``tokens``: ``[..., dim]`` float16, bfloat16 or float32, 1 to 16384 wide (strided tokens are copied); ``weight``
    and ``bias``: ``[dim]`` of one dtype, either may be left out. The statistics, the arithmetic and the
    gradients' sums are float32, each result is rounded once: the output to torch's promotion of the two
    dtypes, the gradients to their inputs' own. The gradient itself has none (no second derivatives).
    """
    if not tokens.is_cuda:
        raise RuntimeError("layer_norm runs on CUDA tensors only (there is no CPU path).")
    if tokens.dtype not in _FLOATS:
        raise ValueError("layer_norm: tokens must be float16, bfloat16 or float32.")
    if tokens.ndim < 1 or not 1 <= tokens.shape[-1] <= LAYER_NORM_MAX_DIM:
        raise ValueError(f"layer_norm: the last dimension must have 1 to {LAYER_NORM_MAX_DIM} values.")
    if not eps >= 0.0:
        raise ValueError("layer_norm: eps must not be negative.")
    given = [gain for gain in (weight, bias) if gain is not None]
    for gain in given:
        if gain.shape != tokens.shape[-1:] or gain.device != tokens.device:
            raise ValueError("layer_norm: weight and bias must be [dim] on the tokens' device.")
        if gain.dtype not in _FLOATS or gain.dtype != given[0].dtype:
            raise ValueError("layer_norm: weight and bias must have one dtype of float16, bfloat16 or float32.")
    _lib.refuse_forward_mode("layer_norm", tokens, *given)
    tokens = tokens.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(tensor.requires_grad for tensor in (tokens, *given)):
        return _LayerNorm.apply(tokens, weight, bias, float(eps))
    return _layer_norm_forward(tokens, weight, bias, float(eps), False)[0]
