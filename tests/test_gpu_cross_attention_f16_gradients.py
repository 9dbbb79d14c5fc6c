"""float16 gradients of the attention to another sequence, far below and above one.

The gradient of a logit, dS = P (dP - delta), is held times a power of two that follows the sizes of dO and V. A gradient that is
a power of two smaller therefore gives the same bits, as long as the results themselves stay normal values of float16.
Against float64 the 2-norm of the difference is at most 8 half steps of the result's: a rounding of dS, one of P (dV), one of the
result, delta through the rounded O (two), each at most a half step of terms that add up with signs, which leaves three for the
exponentials and the f32 sums.
"""

from __future__ import annotations

import pytest
import torch

from moss_image_b200.cross_attention import cross_attention, cross_attention_packed
from moss_image_b200.packed import cumulative_lengths
from moss_image_b200.quant_kernels import check_device_status

pytestmark = pytest.mark.gpu

F16 = torch.float16


def _randn(*shape, seed, size=1.0):
    return (size * torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")).to(F16)


def _coarse(*shape, seed):
    """Gradients of few bits: exact at any of the sizes below."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(-16, 17, shape, generator=gen, device="cuda") / 8).to(F16)


def _gradients(q, k, v, grad, **options):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(cross_attention(*leaves, **options), leaves, grad)
    check_device_status(q.device)
    return got


def _exact(q, k, v, grad):
    """dQ, dK, dV in float64, for [batch, tokens, heads, dim] tensors of one scale head_dim ** -0.5."""
    groups, scale = q.shape[2] // k.shape[2], q.shape[3] ** -0.5
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    a, b, c = (t.transpose(1, 2) for t in leaves)
    p = torch.softmax(scale * (a @ b.repeat_interleave(groups, 1).mT), -1)
    o = (p @ c.repeat_interleave(groups, 1)).transpose(1, 2)
    return torch.autograd.grad(o, leaves, grad.double())


def _near(got, exact):
    return (got.double() - exact).norm() <= 8 * 2.0 ** -11 * exact.norm()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tq,tk", [(150, 4096), (3, 2050), (2048, 70)])
def test_a_smaller_gradient_gives_the_same_bits(cuda_device, tq, tk, dim):
    v, grad = _randn(2, tk, 1, dim, seed=1), _coarse(2, tq, 2, dim, seed=2)
    for q_size, k_size, which in ((2.0 ** -10, 2.0 ** 10, 0), (2.0 ** 10, 2.0 ** -10, 1)):  # so that dQ, or dK, stays normal
        q, k = _randn(2, tq, 2, dim, seed=3, size=q_size), _randn(2, tk, 1, dim, seed=4, size=k_size)
        whole = _gradients(q, k, v, grad)[which]
        exact = _exact(q, k, v, grad)[which]
        assert _near(whole, exact)
        for power in (4, 13):
            small = _gradients(q, k, v, grad * 2.0 ** -power)[which]
            normal = whole.abs().double() * 2.0 ** -power >= 2.0 ** -13  # (a rounded 2^-14 may come from below the normal ones)
            assert normal.double().mean() > 0.25  # there is something to compare
            assert torch.equal(small[normal].double() * 2.0 ** power, whole[normal].double())
            assert _near(small.double() * 2.0 ** power, exact)


def test_rows_of_different_sizes(cuda_device):
    q, k = _randn(1, 300, 2, 64, seed=5, size=2.0 ** -8), _randn(1, 2100, 1, 64, seed=6, size=2.0 ** 8)
    v, grad = _randn(1, 2100, 1, 64, seed=7), _coarse(1, 300, 2, 64, seed=8)
    grad = grad * (2.0 ** -(torch.arange(300, device="cuda") % 13))[None, :, None, None].to(F16)
    dq, _, _ = _gradients(q, k, v, grad)
    exact, _, _ = _exact(q, k, v, grad)
    for at in range(13):  # by the size of their gradients
        assert _near(dq[:, at::13], exact[:, at::13]), at


def test_large_values_do_not_overflow(cuda_device):
    q, k = _randn(1, 200, 1, 64, seed=9, size=2.0 ** -7), _randn(1, 300, 1, 64, seed=10, size=2.0 ** -7)
    v, grad = _randn(1, 300, 1, 64, seed=11, size=2.0 ** 12), _coarse(1, 200, 1, 64, seed=12) * 16
    got, exact = _gradients(q, k, v, grad), _exact(q, k, v, grad)
    assert all(t.isfinite().all() for t in got)
    assert all(_near(a, b) for a, b in zip(got[:2], exact[:2]))


def test_sizes_of_one_sequence_do_not_reach_another(cuda_device):
    """Large, small, infinite and NaN values and gradients of some entries, masked or not, leave the others' bits alone."""
    q, k, v, grad = (_randn(3, n, 2, 64, seed=n) for n in (130, 200, 201, 131))
    v, k = v[:, :200], k[:, :200]
    grad = grad[:, :130] * 2.0 ** -6
    mask = torch.ones(3, 200, dtype=torch.bool, device="cuda")
    mask[:, 150:170] = False
    clean = _gradients(q, k, v, grad, key_mask=mask)
    flat = [t.flatten(0, 1) for t in (q, k, v, grad)]
    offsets = [cumulative_lengths([n] * 3, q.device) for n in (130, 200)]

    def packed(q, k, v, grad):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(cross_attention_packed(*leaves, *offsets), leaves, grad)

    plain = packed(*flat)
    for poison in (6e4, float("inf"), float("nan")):
        bad_v, bad_grad = v.clone(), grad.clone()
        bad_v[:, 150:170] = poison  # masked: no entry sees it
        bad_v[1, 3, 0], bad_grad[1, 7, 0] = poison, poison
        got = _gradients(q, k, bad_v, bad_grad, key_mask=mask)
        for a, b in zip(got, clean):
            assert torch.equal(a[[0, 2]], b[[0, 2]]) and torch.equal(a[1, :, 1], b[1, :, 1])
        bad_v[:, 150:170] = v[:, 150:170]
        for a, b, n in zip(packed(flat[0], flat[1], bad_v.flatten(0, 1), bad_grad.flatten(0, 1)), plain, (130, 200, 200)):
            assert torch.equal(a[:n], b[:n]) and torch.equal(a[2 * n:], b[2 * n:])


def test_small_gradients_in_a_graph(cuda_device):
    q, k, v, grad = (_randn(2, 140, 1, 64, seed=s) for s in range(20, 24))
    first = _gradients(q, k, v, grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _gradients_only(q, k, v, grad)
    v.mul_(2.0 ** 4)
    grad.mul_(2.0 ** -8)
    for _ in range(2):  # what one replay found does not stay for the next
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, _gradients(q, k, v, grad)))
    assert not torch.equal(captured[0], first[0])


def _gradients_only(q, k, v, grad):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(cross_attention(*leaves), leaves, grad)
