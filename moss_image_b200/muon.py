"""Orthogonalised updates of trained matrices on the tensor cores (``moss_orthogonalize``).

For the projections that are trained in full (``full_qkvo`` models) and for adapter factors: the
optimiser replaces a matrix's momentum by the nearest matrix with equal singular values, found by
a few steps of an odd polynomial (Newton-Schulz; the Muon optimiser of Jordan et al., 2024),

    X = G / max(|G|, eps);   A = X X^T,  X <- a X + (b A + c A A) X   (each step)

:func:`orthogonalize` is that map for one matrix or a batch of them, :class:`Muon` the optimiser
around it. CUDA tensors only: there is no CPU path.

The result is bfloat16 whatever the input's type: it is a direction, and its own rounding is the
largest error in it. The iteration runs on float16 operands with float32 sums (float32 throughout
when the shorter side is at most 64), which with the usual coefficients keeps the error against float64
within 1.5 times that rounding. An infinity or NaN in a matrix gives a NaN matrix; a zero matrix gives zeros.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from typing import Iterable, Sequence

import torch

from . import _lib
from .quant_kernels import poll_device_status, status_buffer

# What one call of a step may hold besides the parameters and their state (sums, directions, workspace). Matrices that fill
# the GPU gain nothing from a larger batch: four of 3072 x 3072 take as long a matrix as forty.
STEP_BYTES = 1 << 30
_MOST_MATRICES = 65535  # in one call

# Steep at zero: small singular values grow 3.4-fold a step, and all end within about 0.7 to 1.2.
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


@lru_cache(maxsize=1024)
def _workspace_bytes(device: int, batch: int, rows: int, cols: int) -> int:
    size = ctypes.c_size_t()
    with torch.cuda.device(device):  # the plan counts its multiprocessors
        _lib.check(_lib.library().moss_orthogonalize_workspace_bytes(batch, rows, cols, ctypes.byref(size)),
                   "moss_orthogonalize_workspace_bytes")
    return size.value


def _coefficient_array(coefficients: tuple, steps: int) -> ctypes.Array:
    if coefficients and not isinstance(coefficients[0], tuple):
        coefficients = (coefficients,) * steps
    if len(coefficients) != steps or any(len(step) != 3 for step in coefficients):
        raise ValueError("orthogonalize: coefficients must be (a, b, c), or one such triple for each step.")
    return (ctypes.c_float * (3 * steps))(*(float(value) for step in coefficients for value in step))


@lru_cache(maxsize=64)
def _checked_steps(coefficients: tuple, steps: int, eps: float) -> ctypes.Array:
    if not 1 <= steps <= 16:
        raise ValueError("orthogonalize: steps must be between 1 and 16.")
    if not (eps > 0.0 and math.isfinite(eps)):
        raise ValueError("orthogonalize: eps must be positive and finite.")
    values = _coefficient_array(coefficients, steps)
    # of no matrices: the library looks at the steps and returns
    _lib.check(_lib.library().moss_orthogonalize(None, _lib.DTYPE_CODES[torch.float32], 0, 0, 0, steps, values, eps, None,
                                                 None, 0, None, None), "moss_orthogonalize")
    return values


def _step_values(steps: int, coefficients: Sequence, eps: float) -> ctypes.Array:
    """The coefficients of each step, once all that does not depend on the matrices is checked."""
    if coefficients is not COEFFICIENTS:
        coefficients = tuple(tuple(c) if isinstance(c, (tuple, list)) else c for c in coefficients)
    return _checked_steps(coefficients, steps, float(eps))


class _WithoutGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, update, *options):
        return orthogonalize(update, *options)

    @staticmethod
    def backward(ctx, gradient):
        raise NotImplementedError("orthogonalize has no gradient: detach the update.")


def orthogonalize(update: torch.Tensor, steps: int = 5,
                  coefficients: Sequence[float] | Sequence[Sequence[float]] = COEFFICIENTS, eps: float = 1e-7, *,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The orthogonalised update of ``[rows, cols]`` or each of ``[..., rows, cols]``, in bfloat16.

    ``update``: float16, bfloat16 or float32 on CUDA. ``coefficients``: one ``(a, b, c)`` for all ``steps``
    (1 to 16), or one for each. ``eps``: the least norm a matrix is divided by. Not differentiable: a backward
    pass that reaches an update that requires grad raises.
    """
    if not update.is_cuda:
        raise RuntimeError("orthogonalize runs on CUDA tensors only (there is no CPU path).")
    if update.ndim < 2 or update.dtype not in _lib.DTYPE_CODES:
        raise ValueError("orthogonalize: the update must be a float16, bfloat16 or float32 [..., rows, cols] tensor.")
    _lib.refuse_forward_mode("orthogonalize", update)
    values = _step_values(steps, coefficients, eps)
    if torch.is_grad_enabled() and update.requires_grad:
        if out is not None:
            raise RuntimeError("orthogonalize: an update that requires grad cannot be written to an output buffer.")
        return _WithoutGradient.apply(update, steps, coefficients, eps)
    device = update.device
    if device.index != _lib.current_device_index():
        with torch.cuda.device(device):
            return orthogonalize(update, steps, coefficients, eps, out=out)
    status = status_buffer(device)
    poll_device_status(device)
    update = update.detach().contiguous()
    if out is None:
        out = torch.empty(update.shape, dtype=torch.bfloat16, device=device)
    elif out.shape != update.shape or out.dtype != torch.bfloat16 or out.device != device or not out.is_contiguous():
        raise ValueError("orthogonalize: the output buffer must be a contiguous bfloat16 tensor like the update.")
    rows, cols = update.shape[-2:]
    batch = 1
    for length in update.shape[:-2]:
        batch *= length
    size = _workspace_bytes(device.index, batch, rows, cols)
    workspace = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _lib.check(_lib.library().moss_orthogonalize(
        update.data_ptr(), _lib.DTYPE_CODES[update.dtype], batch, rows, cols, steps, values, float(eps), out.data_ptr(),
        _lib.ptr(workspace), size, status.data_ptr(), _lib.stream_handle(device)), "moss_orthogonalize")
    _lib.count_launch("orthogonalize")
    return out


def _check_options(group: dict) -> None:
    if group["lr"] < 0.0 or group["weight_decay"] < 0.0 or not 0.0 <= group["momentum"] < 1.0:
        raise ValueError("Muon: lr and weight_decay must not be negative, and momentum must be in [0, 1).")
    _step_values(group["steps"], group["coefficients"], group["eps"])


def _matrices_at_once(device: int, rows: int, cols: int) -> int:
    # two sums in float32, the direction in bfloat16
    one = 10 * rows * cols + _workspace_bytes(device, 1, rows, cols)
    side = -(-min(rows, cols) // 128) * 128
    return max(1, min(STEP_BYTES // max(one, 1), _MOST_MATRICES, (2**31 - 1) // max(side, 1)))


class Muon(torch.optim.Optimizer):
    """Momentum, orthogonalised, as the update of each trained matrix.

    ``m <- momentum m + g``; the direction is ``orthogonalize(g + momentum m)`` (``nesterov``) or
    ``orthogonalize(m)``; then ``w <- (1 - lr weight_decay) w - lr s direction`` with
    ``s = 0.2 sqrt(max(rows, cols))``, which gives the update the root mean square that AdamW's usually
    has, so that its learning rates carry over. Matrices only: norms, biases and embeddings
    belong to another optimiser. Parameters of one shape and dtype are orthogonalised together, as many at
    a time as ``STEP_BYTES`` of memory allow.

    The state is float32 whatever the parameters' type. For 16-bit parameters it also holds what their last
    rounding left out (``remainder``): decay and update are applied to the sum of the two, so that steps far
    below half a rounding step of a weight add up. A weight changed from outside keeps its new value.
    """

    def __init__(self, params: Iterable, lr: float = 1e-3, *, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS,
                 eps: float = 1e-7) -> None:
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, param_group: dict) -> None:
        _check_options({**self.defaults, **param_group})
        super().add_param_group(param_group)
        if any(p.ndim != 2 or p.dtype not in _lib.DTYPE_CODES for p in self.param_groups[-1]["params"]):
            self.param_groups.pop()
            raise ValueError("Muon updates matrices only (2 dimensions), of float16, bfloat16 or float32.")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        parts = []  # all that can be refused is, before a parameter or its state changes
        for group in self.param_groups:
            _check_options(group)
            shapes: dict[tuple, list[torch.Tensor]] = {}
            for p in group["params"]:
                if p.grad is not None:
                    shapes.setdefault((p.shape, p.dtype, p.device), []).append(p)
            for (shape, _, device), params in shapes.items():
                if device.type != "cuda":
                    raise RuntimeError("Muon runs on CUDA tensors only (there is no CPU path).")
                most = _matrices_at_once(device.index, *shape)
                parts.extend((group, shape, params[first:first + most]) for first in range(0, len(params), most))
        for part in parts:
            self._step_shape(*part)
        return loss

    def _step_shape(self, group: dict, shape: torch.Size, params: list[torch.Tensor]) -> None:
        momentum, grads = group["momentum"], [p.grad for p in params]
        wide = params[0].dtype == torch.float32
        buffers, remainders = [], []
        for p in params:
            state = self.state[p]
            if "momentum_buffer" not in state:
                state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
            if not wide and "remainder" not in state:
                state["remainder"] = torch.zeros_like(p, dtype=torch.float32)
            buffers.append(state["momentum_buffer"])
            if not wide:
                remainders.append(state["remainder"])
        if wide:
            torch._foreach_mul_(buffers, momentum)
            torch._foreach_add_(buffers, grads)
            updates = torch.stack(torch._foreach_add(grads, buffers, alpha=momentum) if group["nesterov"] else buffers)
        else:
            updates = torch.empty(len(params), *shape, device=params[0].device)
            for grad, buffer, update in zip(grads, buffers, updates):
                torch.add(grad, buffer, alpha=momentum, out=buffer)
                if group["nesterov"]:
                    torch.add(grad, buffer, alpha=momentum, out=update)
                else:
                    update.copy_(buffer)
        directions = orthogonalize(updates, group["steps"], group["coefficients"], group["eps"])
        del updates
        rate = group["lr"] * 0.2 * math.sqrt(max(shape))
        keep = 1.0 - group["lr"] * group["weight_decay"]
        if wide:
            if group["weight_decay"]:
                torch._foreach_mul_(params, keep)
            torch._foreach_add_(params, list(directions.unbind(0)), alpha=-rate)
            return
        for p, remainder, direction in zip(params, remainders, directions):
            held = p.float()
            exact = remainder + held
            # a weight that its remainder no longer rounds to was changed from outside
            exact = torch.where(exact.to(p.dtype) == p, exact, held)
            if group["weight_decay"]:
                exact.mul_(keep)
            exact.add_(direction, alpha=-rate)
            p.copy_(exact)
            torch.sub(exact, p, out=remainder)

    def load_state_dict(self, state_dict: dict) -> None:
        super().load_state_dict(state_dict)
        # the base class casts state to the parameter's type: the float32 state is taken as it was saved
        saved = [index for group in state_dict["param_groups"] for index in group["params"]]
        for index, p in zip(saved, (p for group in self.param_groups for p in group["params"])):
            for name, value in state_dict["state"].get(index, {}).items():
                self.state[p][name] = value.to(device=p.device, dtype=torch.float32, copy=True)
