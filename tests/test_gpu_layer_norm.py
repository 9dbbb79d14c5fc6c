"""Layer norm and its gradients on the GPU against the definition in float64.

Bounds (u = 2^-24): a row's sum is a tree at most D = 57 additions deep (32 values of a thread, 5 shuffles, 16
warps, and the division), so the mean is off by D u mean|x| and the variance by (D + 3) u of itself, the
inverse deviation by half of that and the root's two steps. Everything else is a handful of f32 roundings, and
one rounding to the result's type: half a step.
"""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

from moss_image_b200 import _lib
from moss_image_b200.norms import layer_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DEPTH = 60
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _half_steps(exact: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    # relative to the value; results below the normal range round to a fixed step
    return HALF_STEP[dtype] * exact.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _assert_within(name: str, got: torch.Tensor, exact: torch.Tensor, slack: torch.Tensor) -> None:
    off = (got.double() - exact).abs()
    allowed = slack + _half_steps(exact.abs() + slack, got.dtype)
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of what rounding allows"


def _check(x, weight, bias, grad, eps=1e-6):
    leaves = [t.detach().requires_grad_() for t in (x, weight, bias) if t is not None]
    named = iter(leaves)
    y = layer_norm(next(named), None if weight is None else next(named), None if bias is None else next(named), eps)
    got = torch.autograd.grad(y, leaves, grad)
    xd = x.double()
    dim = x.shape[-1]
    w = torch.ones(dim, device=x.device, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(dim, device=x.device, dtype=torch.float64) if bias is None else bias.double()
    mean = xd.mean(-1, keepdim=True)
    rstd = ((xd - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    n = (xd - mean) * rstd
    dn_off = U * (DEPTH * xd.abs().mean(-1, keepdim=True) * rstd + DEPTH * n.abs())
    _assert_within("y", y.detach(), n * w + b, w.abs() * dn_off + 3 * U * ((n * w).abs() + b.abs()))

    d = grad.double()
    dn = d * w
    s0, s1 = dn.mean(-1, keepdim=True), (dn * n).mean(-1, keepdim=True)
    s1_off = DEPTH * U * (dn * n).abs().mean(-1, keepdim=True) + (dn.abs() * dn_off).mean(-1, keepdim=True)
    parts = dn.abs() + s0.abs() + (n * s1).abs()
    dx_off = rstd * (DEPTH * U * dn.abs().mean(-1, keepdim=True) + n.abs() * s1_off + dn_off * s1.abs() + (DEPTH + 8) * U * parts)
    _assert_within("dx", got[0], rstd * (dn - s0 - n * s1), dx_off)
    flat = [t.reshape(-1, dim) for t in (d, n, dn_off)]
    # a column's sum: the rows of one team, up to 64 teams, a run of partials and eight runs
    depth = x[..., 0].numel() / 148 + 2 + 64 + 19 + 8
    at = 1
    if weight is not None:
        terms = (flat[0] * flat[1]).abs().sum(0)
        _assert_within("dw", got[at], (flat[0] * flat[1]).sum(0), depth * U * terms + (flat[0].abs() * flat[2]).sum(0))
        at += 1
    if bias is not None:
        _assert_within("db", got[at], flat[0].sum(0), depth * U * flat[0].abs().sum(0))
    return y, got


def _inputs(shape, dtype, gain, seed, offset=0.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dim = shape[-1]

    def randn(*size):
        return torch.randn(*size, generator=gen, device="cuda")

    x = (randn(*shape) * torch.exp(0.5 * randn(dim)) + offset * randn(dim)).to(dtype)
    gain_dtype = {"same": dtype, "f32": F32, "none": None}[gain]
    weight = bias = None
    if gain_dtype is not None:
        weight, bias = (1 + 0.2 * randn(dim)).to(gain_dtype), (0.1 * randn(dim)).to(gain_dtype)
    out_dtype = dtype if gain_dtype is None else torch.promote_types(dtype, gain_dtype)
    return x, weight, bias, (1e-1 * randn(*shape)).to(out_dtype)


# widths around every change of team and vector: 8, 32, 128 and 512 threads with vectors of 8, 2 and 1
WIDTHS = [1, 2, 7, 8, 17, 192, 200, 512, 514, 768, 776, 1090, 2047, 2050, 3072, 3080, 8191, 12288, 12296, 16383, 16384]


@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("dtype,gain", [(BF16, "same"), (F16, "f32"), (F32, "same"), (BF16, "none")])
def test_matches_the_definition(cuda_device, dim, dtype, gain):
    _check(*_inputs((5 if dim > 4096 else 67, dim), dtype, gain, dim))


@pytest.mark.parametrize("rows,dim,dtype,gain", [(1, 64, BF16, "same"), (4099, 96, F16, "same"), (2500, 768, BF16, "f32"),
                                                 (1777, 1090, F16, "same"), (700, 4096, F32, "none")])
def test_more_rows_than_teams(cuda_device, rows, dim, dtype, gain):
    _check(*_inputs((rows, dim), dtype, gain, rows))


def test_leading_dimensions_strides_and_alignment(cuda_device):
    x, weight, bias, grad = _inputs((3, 5, 7, 48), BF16, "same", 1)
    _check(x, weight, bias, grad)
    fused = torch.randn(11, 4, 3, 64, device="cuda").to(BF16)
    view = fused[:, :, 1]  # not dense: copied
    _check(view, weight[:1].expand(64), bias[:1].expand(64), torch.randn(11, 4, 64, device="cuda").to(BF16))
    flat = torch.randn(1 + 9 * 64, device="cuda").to(F16)
    offset = flat[1:].view(9, 64)  # dense rows off the 16-byte grid: narrower vectors
    assert offset.data_ptr() % 16 == 2
    gains = torch.randn(65, device="cuda").to(F16)
    _check(offset, gains[1:], gains[:64], torch.randn(9, 64, device="cuda").to(F16))


def test_one_of_gain_and_offset(cuda_device):
    x, weight, bias, grad = _inputs((33, 320), BF16, "same", 2)
    _check(x, weight, None, grad)
    _check(x, None, bias, grad)


def test_means_far_from_zero_and_constant_rows(cuda_device):
    x, weight, bias, grad = _inputs((16, 1000), F32, "same", 3)
    _check(x + 3000.0, weight, bias, grad)
    y = layer_norm(torch.full((4, 24), 7.0, device="cuda", dtype=BF16), weight[:24].to(BF16), bias[:24].to(BF16))
    assert torch.equal(y, bias[:24].to(BF16).expand(4, 24))


def test_non_finite_rows_stay_alone(cuda_device):
    x, weight, bias, grad = _inputs((40, 96), F16, "same", 4)
    clean = layer_norm(x, weight, bias)
    x[7, 3], x[21, 50] = float("nan"), float("inf")
    y = layer_norm(x, weight, bias)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 21]] = True
    assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])


def test_no_rows(cuda_device):
    x = torch.empty(0, 72, device="cuda", dtype=BF16, requires_grad=True)
    weight, bias = (torch.ones(72, device="cuda", dtype=BF16, requires_grad=True) for _ in range(2))
    y = layer_norm(x, weight, bias)
    dx, dw, db = torch.autograd.grad(y, (x, weight, bias), torch.empty_like(y))
    assert y.shape == dx.shape == (0, 72) and not dw.any() and not db.any()


def test_only_the_gradients_that_are_asked_for(cuda_device):
    x, weight, bias, grad = _inputs((50, 200), BF16, "same", 5)
    _, full = _check(x, weight, bias, grad)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, weight, bias))]
        y = layer_norm(*leaves)
        for i, part in zip(wanted, torch.autograd.grad(y, [leaves[i] for i in wanted], grad)):
            assert torch.equal(part, full[i])


def test_gradient_against_differences(cuda_device):
    x, weight, bias, grad = _inputs((6, 40), F32, "same", 6)
    _, got = _check(x, weight, bias, grad)

    def loss(*values):
        return (torch.nn.functional.layer_norm(values[0], (40,), values[1], values[2], 1e-6) * grad.double()).sum()

    points = [t.double() for t in (x, weight, bias)]
    for i, part in enumerate(got):
        step = torch.randn_like(points[i])
        h = 1e-5
        moved = [[p + s * h * step if k == i else p for k, p in enumerate(points)] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * h)
        # the slope: central differences, off by h^2 times third derivatives; the gradient: f32 rounding
        assert abs((part.double() * step).sum() - slope) <= 1e-5 * (part.double() * step).abs().sum()


def test_same_bits_every_time_on_a_side_stream_and_in_a_graph(cuda_device):
    x, weight, bias, grad = _inputs((3001, 640), BF16, "same", 7)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, weight, bias)]
        y = layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, grad)]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    x.copy_(x.flip(0))
    grad.copy_(grad.flip(0))
    graph.replay()
    assert all(torch.equal(a, b.flip(0)) for a, b in zip(first[:2], captured[:2]))
    fresh = step()
    assert all(torch.equal(a, b) for a, b in zip(fresh, captured))


def test_refusals(cuda_device):
    x = torch.randn(4, 32, device="cuda", dtype=BF16)
    weight = torch.ones(32, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="one dtype"):
        layer_norm(x, weight, weight.float())
    with pytest.raises(ValueError, match="dim"):
        layer_norm(x, weight[:31])
    with pytest.raises(ValueError, match="device"):
        layer_norm(x, weight.cpu())
    with pytest.raises(ValueError, match="float16"):
        layer_norm(x.double())
    with pytest.raises(ValueError, match="16384"):
        layer_norm(torch.empty(2, 16385, device="cuda"))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, eps=-1.0)
    leaf = x.detach().requires_grad_()
    slope, = torch.autograd.grad(layer_norm(leaf).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(slope.float().sum(), leaf)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            layer_norm(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("dims", [(6144, 12288), (1024, 3072)])
def test_two_threads_at_once(cuda_device, dims):
    """Widths that run the same kernels with different shared memory, from two threads on streams of their own."""
    cases = []
    for dim in dims:
        x, weight, bias, grad = _inputs((8, dim), BF16, "same", dim)
        y, (dx, dw, db) = _check(x, weight, bias, grad)
        cases.append((x, weight, bias, grad, y.detach(), dx, dw, db))
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(cases)), []

    def run(x, weight, bias, grad, *expected):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                rows, dim = x.shape
                got = [torch.empty_like(t) for t in expected]
                stats = torch.empty(rows, 2, device="cuda")
                size = ctypes.c_size_t()
                lib, stream = _lib.library(), torch.cuda.current_stream().cuda_stream
                _lib.check(lib.moss_layernorm_bwd_workspace_bytes(rows, dim, ctypes.byref(size)), "workspace")
                workspace = torch.empty(size.value, dtype=torch.uint8, device="cuda")
                forward = (x.data_ptr(), 1, rows, dim, weight.data_ptr(), bias.data_ptr(), 1, 1e-6, got[0].data_ptr(),
                           stats.data_ptr(), stream)
                backward = (grad.data_ptr(), x.data_ptr(), 1, rows, dim, weight.data_ptr(), 1, stats.data_ptr(), 1,
                            *(t.data_ptr() for t in got[1:]), workspace.data_ptr(), size.value, stream)
                start.wait()
                for _ in range(20000):  # the entry points themselves, as close together as they come
                    _lib.check(lib.moss_layernorm_fwd(*forward), "moss_layernorm_fwd")
                    _lib.check(lib.moss_layernorm_bwd(*backward), "moss_layernorm_bwd")
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, expected))
        except Exception as error:  # (the test's own thread tells it)
            wrong.append(error)

    threads = [threading.Thread(target=run, args=case) for case in cases]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong, wrong[0]
