"""Rotary positions of queries and keys on the native kernel (``moss_rotary``).

The reference block turns q and k by their positions between the per-head norms and the
attention (training/model.py:269-314). :func:`apply_rotary` does both tensors in one launch, in
the interleaved layout (pairs ``2i, 2i + 1``) or the half layout (pairs ``i, i + R / 2``), over the
whole head or its first ``R`` values, and its gradient is the same kernel with the angles
negated. :func:`rotary_frequencies` and :func:`rotary_table` make the angles, once for all blocks
of a step; they are plain torch in float64, so that large positions keep their angle.

CUDA tensors only for :func:`apply_rotary`: there is no CPU path.
"""

from __future__ import annotations

import math
from typing import Sequence

import torch

from . import _lib

_SCALINGS = (None, "linear", "ntk", "yarn")


def rotary_frequencies(dim: int, *, theta: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device: torch.device | str | None = None) -> torch.Tensor:
    """Angle per position of each pair of ``dim`` rotated values: float64 ``[dim / 2]``.

    ``scaling`` stretches the positions by ``factor`` for sequences longer than the trained ones:
    ``"linear"`` divides every frequency by it; ``"ntk"`` raises the base so that only the slowest
    frequency is divided by it; ``"yarn"`` (Peng et al., 2023) divides the pairs that turn fewer than
    ``beta_slow`` times over ``original_length`` positions, keeps those that turn more than
    ``beta_fast`` times, and blends in between (see :func:`yarn_magnitude` for its gain).
    """
    if dim < 2 or dim % 2 != 0:
        raise ValueError("rotary dim must be even and positive.")
    if scaling not in _SCALINGS:
        raise ValueError("rotary scaling must be None, 'linear', 'ntk' or 'yarn'.")
    if not theta > 0.0 or not factor >= 1.0:
        raise ValueError("rotary theta must be positive and factor at least 1.")
    exponent = torch.arange(dim // 2, dtype=torch.float64, device=device) / (dim // 2)
    if scaling == "ntk" and dim > 2:
        theta = theta * factor ** (dim / (dim - 2))
    frequencies = theta ** -exponent
    if scaling == "linear":
        return frequencies / factor
    if scaling == "yarn":
        if original_length is None or original_length < 1:
            raise ValueError("yarn scaling needs the original_length of the trained positions.")
        # linear in the pair's index between the indexes at which the turns pass the two betas
        def index_of(beta: float) -> float:
            return (dim // 2) * math.log(original_length / (beta * 2.0 * math.pi)) / math.log(theta)

        # (the end may lie past the last pair: every pair then turns often enough to keep a part of its frequency)
        low, high = max(math.floor(index_of(beta_fast)), 0), math.ceil(index_of(beta_slow))
        index = torch.arange(dim // 2, dtype=torch.float64, device=device)
        blend = ((index - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        return frequencies * (1.0 - blend) + frequencies / factor * blend
    return frequencies


def yarn_magnitude(factor: float) -> float:
    """The gain YaRN puts on cos and sin (so that attention logits grow by its square)."""
    return 1.0 if factor <= 1.0 else 0.1 * math.log(factor) + 1.0


def rotary_table(positions: torch.Tensor, frequencies: torch.Tensor | Sequence[torch.Tensor], *,
                 magnitude: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin, float32 ``[tokens, R / 2]``, of the angles ``position * frequency``.

    ``positions`` is ``[tokens]`` with one frequency vector, or ``[tokens, axes]`` with one vector for
    each axis (an image token's frame, row and column), whose pairs follow one another.
    """
    if isinstance(frequencies, torch.Tensor):
        frequencies = (frequencies,)
    places = positions.to(torch.float64)
    if places.ndim == 1:
        places = places[:, None]
    if places.ndim != 2 or places.shape[1] != len(frequencies):
        raise ValueError("rotary positions must be [tokens] or [tokens, axes] with one frequency vector per axis.")
    angles = torch.cat([places[:, axis, None] * vector.to(places)[None] for axis, vector in enumerate(frequencies)], 1)
    return (angles.cos() * magnitude).float(), (angles.sin() * magnitude).float()


def _heads_view(name: str, tensor: torch.Tensor) -> torch.Tensor:
    if tensor.ndim == 3:
        tensor = tensor.unsqueeze(0)
    if tensor.ndim != 4:
        raise ValueError(f"apply_rotary: {name} must be [batch, tokens, heads, head_dim] or [tokens, heads, head_dim].")
    return tensor if tensor.stride(3) == 1 else tensor.contiguous()


def _launch(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None,
            interleaved: bool, inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    device = q.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return _launch(q, k, cos, sin, positions, interleaved, inverse)
    q4, k4 = _heads_view("q", q), _heads_view("k", k)
    batch, tokens, q_heads, head_dim = q4.shape
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    qs, ks = q4.stride(), k4.stride()
    rc = _lib.library().moss_rotary(
        q4.data_ptr(), qs[0], qs[1], qs[2], q_heads, k4.data_ptr(), ks[0], ks[1], ks[2], k4.shape[2],
        _lib.DTYPE_CODES[q.dtype], batch, tokens, head_dim, cos.data_ptr(), sin.data_ptr(), cos.shape[0],
        2 * cos.shape[1], None if positions is None else positions.data_ptr(),
        tokens if positions is not None and positions.ndim == 2 else 0, int(interleaved), int(inverse),
        q_out.data_ptr(), k_out.data_ptr(), _lib.stream_handle(device))
    _lib.check(rc, "moss_rotary")
    _lib.count_launch("rotary")
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved, inverse):
        ctx.save_for_backward(cos, sin, positions)
        ctx.interleaved, ctx.inverse = interleaved, inverse
        return _launch(q, k, cos, sin, positions, interleaved, inverse)

    @staticmethod
    def backward(ctx, q_grad, k_grad):
        cos, sin, positions = ctx.saved_tensors
        _lib.refuse_forward_mode("apply_rotary", q_grad, k_grad)
        # a linear map: its gradient is the opposite turn, and so on for the gradient's
        turn = _Rotary.apply if torch.is_grad_enabled() else _launch
        q_grad, k_grad = turn(q_grad, k_grad, cos, sin, positions, ctx.interleaved, not ctx.inverse)
        return q_grad, k_grad, None, None, None, None, None


def apply_rotary(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *, interleaved: bool = True,
                 positions: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Queries and keys turned by their positions; differentiable in ``q`` and ``k`` (reverse mode, to any order).

    ``q``: ``[batch, tokens, q_heads, head_dim]``, ``k``: the same with its own head count (any strides with
    a dense last dimension; views of a fused projection are read in place), or both packed as
    ``[tokens, heads, head_dim]``; float16, bfloat16 or float32. ``cos``/``sin``: float32 ``[rows, R / 2]`` with
    ``R <= head_dim``; values past ``R`` are copied. Token ``t`` takes row ``t``, or row
    ``positions[t]`` / ``positions[batch, t]`` (int64) of a longer table. The tensors stay on the device
    unread, so a position outside the table is not an error here: its token's turned values come out NaN.
    """
    if not q.is_cuda:
        raise RuntimeError("apply_rotary runs on CUDA tensors only (there is no CPU path).")
    device = q.get_device()
    if k.get_device() != device or cos.get_device() != device or sin.get_device() != device:
        raise ValueError("apply_rotary: q, k, cos and sin must be on one device.")
    if q.dtype != k.dtype or q.dtype not in _lib.DTYPE_CODES:
        raise ValueError("apply_rotary: q and k must have one dtype of float16, bfloat16 or float32.")
    q_shape, k_shape = q.shape, k.shape
    if q.ndim not in (3, 4) or q.ndim != k.ndim or q_shape[:-2] != k_shape[:-2] or q_shape[-1] != k_shape[-1]:
        raise ValueError("apply_rotary: q and k must agree in all dimensions but the heads.")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.ndim != 2 or cos.shape != sin.shape:
        raise ValueError("apply_rotary: cos and sin must be float32 [rows, rotary_dim / 2].")
    if 2 * cos.shape[1] > q_shape[-1]:
        raise ValueError("apply_rotary: the table turns more values than a head has.")
    tokens = q_shape[-3]
    if positions is None:
        if cos.shape[0] < tokens:
            raise ValueError("apply_rotary: the table has fewer rows than there are tokens.")
    else:
        if positions.get_device() != device or positions.dtype != torch.int64:
            raise ValueError("apply_rotary: positions must be int64 on the tensors' device.")
        if tuple(positions.shape) not in ((tokens,), tuple(q_shape[:-2])):
            raise ValueError("apply_rotary: positions must be [tokens] or [batch, tokens].")
        positions = positions.contiguous()
    tracking = torch.is_grad_enabled()
    if tracking and (cos.requires_grad or sin.requires_grad):
        raise ValueError("apply_rotary: the tables get no gradient: detach them.")
    _lib.refuse_forward_mode("apply_rotary", q, k, cos, sin)
    cos, sin = cos.contiguous(), sin.contiguous()
    if tracking and (q.requires_grad or k.requires_grad):
        return _Rotary.apply(q, k, cos, sin, positions, interleaved, False)
    return _launch(q, k, cos, sin, positions, interleaved, False)
