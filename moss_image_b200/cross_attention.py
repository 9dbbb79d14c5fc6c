"""Attention of one sequence's queries to another's keys on the native tensor-core kernels.

The text branch of a block whose image tokens look at a caption: keys and values come from an encoder's
states, of another length than the queries, with captions of several lengths in one batch. Everything runs
in one pass over the keys per query tile (running maximum and sum), nothing of size queries x keys is
written, and the backward pass recomputes the probabilities from the row sums that the forward one keeps.

* :func:`cross_attention`: ``[batch, tokens, heads, head_dim]`` tensors, as the projections and
  :func:`~moss_image_b200.rotary.apply_rotary` leave them, optionally with a mask of the keys.
* :func:`cross_attention_packed`: packed rows of several sequences (:mod:`moss_image_b200.packed`) with
  boundaries for the queries and for the keys, each sequence looking at its own keys.

A query without keys (an empty caption, a mask that leaves nothing, logits of minus infinity) gives zeros, and no
gradient. What lies in masked places is never read into a result, infinities and NaN included; NaN in a place that
is looked at reaches all that depends on it. Gradients of shared key heads and all other sums are float32 in a fixed
order, rounded once. Probabilities and the logits' gradients are rounded to the inputs' type before their products
(float16: times a power of two that keeps them normal); logits are float32, whose own steps show past 2^20.

CUDA tensors only: there is no CPU path.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .quant_kernels import _poll_after_backward, poll_device_status, status_buffer

MAX_HEAD_DIM = 128


def _rows_view(tensor: torch.Tensor) -> torch.Tensor:
    """The tensor as the kernels read it: dense heads, other strides on 16 bytes (a copy where it is not like that)."""
    ok = tensor.stride(-1) == 1 and tensor.data_ptr() % 16 == 0
    for size, stride in zip(tensor.shape[:-1], tensor.stride()[:-1]):
        ok = ok and (size <= 1 or (stride > 0 and stride % 8 == 0))
    return tensor if ok else tensor.clone(memory_format=torch.contiguous_format)


def _strides(tensor: torch.Tensor) -> tuple[int, int, int]:
    return (0, *tensor.stride()[:2]) if tensor.ndim == 3 else tensor.stride()[:3]


@lru_cache(maxsize=1024)
def _workspace_bytes(device: int, *sizes: int) -> int:
    size = ctypes.c_size_t()
    with torch.cuda.device(device):  # the plan counts its multiprocessors
        _lib.check(_lib.library().moss_cross_attention_workspace_bytes(*sizes, ctypes.byref(size)),
                   "moss_cross_attention_workspace_bytes")
    return size.value


def _sizes(q, k, q_offsets) -> tuple[int, int, int, int, int, int, int]:
    """batch, query tokens, key tokens, query heads, key heads, head_dim, packed."""
    if q_offsets is not None:
        return q_offsets.shape[0] - 1, q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], 1
    return q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], 0


def _forward(q, k, v, q_offsets, k_offsets, mask, scale, keep_sums):
    device = q.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return _forward(q, k, v, q_offsets, k_offsets, mask, scale, keep_sums)
    status = status_buffer(device)
    poll_device_status(device)
    sizes = _sizes(q, k, q_offsets)
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    lse = torch.empty(sizes[3], math.prod(q.shape[:-2]), dtype=torch.float32, device=device) if keep_sums else None
    size = _workspace_bytes(device.index, *sizes, 0)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.check(_lib.library().moss_cross_attention_fwd(
        q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v), _lib.DTYPE_CODES[q.dtype],
        *sizes[:6], _lib.ptr(q_offsets), _lib.ptr(k_offsets), _lib.ptr(mask), 0 if mask is None else mask.stride(0), scale,
        out.data_ptr(), _lib.ptr(lse), _lib.ptr(workspace), size, status.data_ptr(), _lib.stream_handle(device)),
        "moss_cross_attention_fwd")
    _lib.count_launch("cross_attention")
    return out, lse


def _backward(grad, q, k, v, q_offsets, k_offsets, mask, scale, out, lse, keys_too):
    device = q.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return _backward(grad, q, k, v, q_offsets, k_offsets, mask, scale, out, lse, keys_too)
    status = status_buffer(device)
    poll_device_status(device)
    sizes = _sizes(q, k, q_offsets)
    grad = grad.contiguous()
    if grad.data_ptr() % 16:
        grad = grad.clone()
    dq = torch.empty(q.shape, dtype=q.dtype, device=device)
    dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=device) if keys_too else None for _ in range(2))
    size = _workspace_bytes(device.index, *sizes, 1)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.check(_lib.library().moss_cross_attention_bwd(
        grad.data_ptr(), q.data_ptr(), *_strides(q), k.data_ptr(), *_strides(k), v.data_ptr(), *_strides(v),
        _lib.DTYPE_CODES[q.dtype], *sizes[:6], _lib.ptr(q_offsets), _lib.ptr(k_offsets), _lib.ptr(mask),
        0 if mask is None else mask.stride(0), scale, out.data_ptr(), lse.data_ptr(), dq.data_ptr(), _lib.ptr(dk),
        _lib.ptr(dv), _lib.ptr(workspace), size, status.data_ptr(), _lib.stream_handle(device)), "moss_cross_attention_bwd")
    _lib.count_launch("cross_attention")
    return dq, dk, dv


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, mask, scale):
        q, k, v = _rows_view(q), _rows_view(k), _rows_view(v)
        out, lse = _forward(q, k, v, q_offsets, k_offsets, mask, scale, True)
        ctx.save_for_backward(q, k, v, q_offsets, k_offsets, mask, out, lse)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, grad):
        # (the guard against second derivatives costs microseconds, and is needed where a graph is recorded)
        return _gradients_once(ctx, grad) if torch.is_grad_enabled() else _gradients(ctx, grad)


def _gradients(ctx, grad):
    q, k, v, q_offsets, k_offsets, mask, out, lse = ctx.saved_tensors
    _lib.refuse_forward_mode("cross_attention", grad)
    _poll_after_backward(grad.device)
    wanted = ctx.needs_input_grad
    dq, dk, dv = _backward(grad, q, k, v, q_offsets, k_offsets, mask, ctx.scale, out, lse, wanted[1] or wanted[2])
    return dq if wanted[0] else None, dk if wanted[1] else None, dv if wanted[2] else None, None, None, None, None


_gradients_once = once_differentiable(_gradients)


def _attend(q, k, v, q_offsets, k_offsets, mask, scale):
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, q_offsets, k_offsets, mask, scale)
    q, k, v = _rows_view(q), _rows_view(k), _rows_view(v)
    return _forward(q, k, v, q_offsets, k_offsets, mask, scale, False)[0]


def _check(q, k, v, ndim, scale, what) -> float:
    if not q.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA tensors only (there is no CPU path).")
    layout = "[batch, tokens, heads, head_dim]" if ndim == 4 else "[tokens, heads, head_dim]"
    if q.ndim != ndim or k.ndim != ndim or v.ndim != ndim:
        raise ValueError(f"{what}: query, key and value must be {layout}.")
    if k.device != q.device or v.device != q.device:
        raise ValueError(f"{what}: query, key and value must be on one device.")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: query, key and value must have one dtype of float16 or bfloat16.")
    if k.shape != v.shape or q.shape[-1] != k.shape[-1] or (ndim == 4 and q.shape[0] != k.shape[0]):
        raise ValueError(f"{what}: key and value must have one shape, with the query's batch and head_dim.")
    heads, shared, dim = q.shape[-2], k.shape[-2], q.shape[-1]
    if not heads or not shared or heads % shared:
        raise ValueError(f"{what}: the query's heads must be a multiple of the key's.")
    if dim % 8 or not 8 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"{what}: head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}.")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"{what}: the scale must be positive and finite.")
    _lib.refuse_forward_mode(what, q, k, v)
    return scale


def cross_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *, key_mask: torch.Tensor | None = None,
                    scale: float | None = None) -> torch.Tensor:
    """``softmax(scale Q K^T) V`` of ``[batch, q_tokens, q_heads, head_dim]`` queries and
    ``[batch, k_tokens, k_heads, head_dim]`` keys and values; differentiable in all three (once).

    float16 or bfloat16, ``head_dim`` a multiple of 8 up to 128, ``q_heads`` a multiple of ``k_heads`` (each key head
    serves that many query heads in a row). Views with dense heads and strides on 16 bytes are read in
    place, others copied. ``key_mask``: bool ``[batch, k_tokens]``, true where a key may be looked at.
    ``scale`` is ``head_dim ** -0.5`` by default.
    """
    what = "cross_attention"
    scale = _check(query, key, value, 4, scale, what)
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape != key.shape[:2] or key_mask.device != query.device:
            raise ValueError(f"{what}: key_mask must be bool [batch, k_tokens] on the query's device.")
        if key_mask.stride(-1) != 1 and key_mask.shape[-1] > 1:
            key_mask = key_mask.contiguous()
    return _attend(query, key, value, None, None, key_mask, scale)


def cross_attention_packed(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, q_offsets: torch.Tensor,
                           k_offsets: torch.Tensor, *, scale: float | None = None) -> torch.Tensor:
    """:func:`cross_attention` over packed sequences: ``[q_total, q_heads, head_dim]`` queries and
    ``[k_total, k_heads, head_dim]`` keys and values, sequence ``s`` holding rows ``q_offsets[s]`` to
    ``q_offsets[s + 1]`` of the queries and ``k_offsets[s]`` to ``k_offsets[s + 1]`` of the keys.

    The boundaries are int64 ``[sequences + 1]`` on the tensors' device, start at 0 and do not decrease; they stay there
    unread. Sequences may be empty on either side. Rows behind the last sequence belong to none: their output and their
    gradients are zeros.
    """
    what = "cross_attention_packed"
    scale = _check(query, key, value, 3, scale, what)
    for offsets in (q_offsets, k_offsets):
        if offsets.dtype != torch.int64 or offsets.ndim != 1 or offsets.device != query.device:
            raise ValueError(f"{what}: offsets must be int64 [sequences + 1] on the query's device.")
    if q_offsets.shape != k_offsets.shape or q_offsets.shape[0] < 2:
        raise ValueError(f"{what}: queries and keys must have the boundaries of the same sequences, one at least.")
    return _attend(query, key, value, q_offsets.contiguous(), k_offsets.contiguous(), None, scale)
