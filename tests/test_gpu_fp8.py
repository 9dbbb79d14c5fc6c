"""The block-scaled fp8 linear on the GPU against its definition in float64."""

from __future__ import annotations

import pytest
import torch
from torch import nn

from moss_image_b200 import fp8
from moss_image_b200.lora import LoRALinear

pytestmark = pytest.mark.gpu

# one rounding to the type (unit roundoff) and half a subnormal step
ROUNDING = {torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float16: (2.0 ** -11, 2.0 ** -25),
            torch.float32: (2.0 ** -24, 2.0 ** -149)}
# Codes have 4 significant bits, so products are exact; a block adds 128 of them in f32, each
# addition off by at most 2^-23 of the terms' magnitude, and the blocks' sums add far less.
SUM_ROOM = 2.0 ** -16


def _round_e4m3(v: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, ties to even, in float64: 3 fraction bits down to 2^-6, then steps of 2^-9."""
    exponent = torch.frexp(v.abs())[1].sub(1).clamp_min(-6).double()
    step = torch.exp2(exponent - 3)
    return ((v / step).round() * step).clamp(-448.0, 448.0)


def _quantized_rows(x: torch.Tensor) -> torch.Tensor:
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[1], 128):
        v = x[:, at : at + 128].double()
        scale = torch.exp2(torch.log2(v.abs().amax(1, keepdim=True).clamp_min(2.0 ** -100) / 448.0).ceil())
        out[:, at : at + 128] = _round_e4m3(v / scale) * scale
    return out


def _decoded(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    n, k = codes.shape
    return codes.float().double() * scale.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _problem(m, k, n, dtype, device, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed + 7 * m + k + n)
    x = (torch.randn(m, k, generator=gen, device=device) * torch.exp(torch.randn(1, k, generator=gen, device=device))).to(dtype)
    weight = torch.randn(n, k, generator=gen, device=device) * torch.exp(torch.randn(n, 1, generator=gen, device=device))
    codes, scale = fp8.quantize_fp8_weight(0.02 * weight)
    bias = torch.randn(n, generator=gen, device=device).to(dtype)
    grad = (1e-2 * torch.randn(m, n, generator=gen, device=device)).to(dtype)
    return x, codes, scale, bias, grad


def _check(got, left, right, bias=None):
    want = left @ right
    size = left.abs() @ right.abs()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    relative, absolute = ROUNDING[got.dtype]
    assert got.shape == want.shape
    assert bool(((got.double() - want).abs() <= relative * want.abs() + absolute + SUM_ROOM * size).all())


SHAPES = [
    (1, 128, 128), (1, 1, 1), (2, 3072, 1030), (16, 640, 384), (17, 200, 300), (33, 1088, 129), (64, 4000, 130),
    (65, 127, 257), (128, 1024, 512), (200, 2050, 1003), (300, 96, 2000), (1030, 640, 2304), (2500, 517, 2049),
    (4096, 256, 1280),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_forward_and_input_gradient(cuda_device, dtype, m, k, n):
    x, codes, scale, bias, grad = _problem(m, k, n, dtype, cuda_device)
    weight = _decoded(codes, scale)
    _check(fp8.fp8_linear_forward(x, codes, scale, bias), _quantized_rows(x), weight.t(), bias)
    _check(fp8.fp8_linear_forward(x, codes, scale), _quantized_rows(x), weight.t())
    _check(fp8.fp8_linear_backward(grad, codes, scale), _quantized_rows(grad), weight)


@pytest.mark.parametrize("m", [3, 96, 700])
def test_float32_in_and_out_and_repeat(cuda_device, m):
    x, codes, scale, bias, _ = _problem(m, 384, 520, torch.float32, cuda_device)
    y = fp8.fp8_linear_forward(x, codes, scale, bias)
    _check(y, _quantized_rows(x), _decoded(codes, scale).t(), bias)
    assert torch.equal(y, fp8.fp8_linear_forward(x, codes, scale, bias))
    half = fp8.fp8_linear_forward(x, codes, scale, bias, torch.bfloat16)
    assert torch.equal(half, y.bfloat16())


def test_row_codes_are_exact(cuda_device):
    """Ties, subnormal codes, the format's ends, empty blocks and blocks below the floor."""
    rows = torch.zeros(8, 256)
    steps = torch.tensor([1.0, 1.0625, 1.125, 1.1875, 1.3125, 1.9375, 0.015625, 0.0009765625, 0.0029296875, 1.75])
    rows[0, : len(steps)] = steps
    rows[1, :128] = torch.linspace(-1.0, 1.0, 128)
    rows[2, 0], rows[2, 128] = 448.0, 449.0
    rows[3, 5], rows[3, 130] = 3.0e38, -1.0e-38
    rows[4, :] = 2.0 ** -101
    rows[5, 7] = 1.7500001
    rows[6, 200] = -2.0 ** -60
    x = rows.to(cuda_device)
    codes, scale = fp8.quantize_fp8_rows(x)
    assert torch.equal(torch.exp2(torch.log2(scale).round()), scale)
    decoded = codes.float().double() * scale.double().repeat_interleave(128, 1)
    assert torch.equal(decoded, _quantized_rows(x))
    assert float(scale[2, 0]) == 1.0 and float(scale[2, 1]) == 2.0 and float(scale[7, 0]) == 2.0 ** -108


def test_weight_codes_match_the_definition(cuda_device):
    gen = torch.Generator().manual_seed(1)
    weight = (torch.randn(300, 200, generator=gen) * 0.02).to(cuda_device)
    codes, scale = fp8.quantize_fp8_weight(weight)
    padded = torch.zeros(384, 256, device=cuda_device)
    padded[:300, :200] = weight
    blocks = padded.view(3, 128, 2, 128)
    want_scale = (blocks.abs().amax((1, 3)).double() / 448.0).float()  # torch multiplies by 1 / 448 in float32
    want = (blocks / want_scale[:, None, :, None]).view(384, 256)[:300, :200].to(torch.float8_e4m3fn)
    assert torch.equal(scale, want_scale)
    assert torch.equal(codes.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))
    weight[5, 5] = float("nan")
    with pytest.raises(ValueError, match="non-finite"):
        fp8.quantize_fp8_weight(weight)


@pytest.mark.parametrize("m", [5, 90, 600])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_nonfinite_value_shows_in_its_row_only(cuda_device, m, value):
    x, codes, scale, _, grad = _problem(m, 300, 260, torch.bfloat16, cuda_device)
    clean, clean_grad = fp8.fp8_linear_forward(x, codes, scale), fp8.fp8_linear_backward(grad, codes, scale)
    x[3, 140], grad[1, 0] = value, value
    y, dx = fp8.fp8_linear_forward(x, codes, scale), fp8.fp8_linear_backward(grad, codes, scale)
    keep = torch.arange(m, device=cuda_device)
    assert y[3].isnan().all() and torch.equal(y[keep != 3], clean[keep != 3])
    assert dx[1].isnan().all() and torch.equal(dx[keep != 1], clean_grad[keep != 1])


def test_zero_rows_and_tiny_gradients(cuda_device):
    _, codes, scale, _, _ = _problem(4, 256, 256, torch.bfloat16, cuda_device)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=cuda_device)
    assert not fp8.fp8_linear_forward(x, codes, scale).any()
    grad = torch.full((4, 256), 1e-20, dtype=torch.bfloat16, device=cuda_device)
    _check(fp8.fp8_linear_backward(grad, codes, scale), _quantized_rows(grad), _decoded(codes, scale))


def test_leading_dimensions_strides_streams_and_empty(cuda_device):
    x, codes, scale, bias, _ = _problem(12, 96, 80, torch.bfloat16, cuda_device)
    y = fp8.fp8_linear_forward(x, codes, scale, bias)
    assert torch.equal(fp8.fp8_linear_forward(x.view(3, 4, 96), codes, scale, bias), y.view(3, 4, 80))
    assert torch.equal(fp8.fp8_linear_forward(x.t().contiguous().t(), codes, scale, bias), y)
    assert torch.equal(fp8.fp8_linear_forward(x[0], codes, scale, bias), y[0])
    out = torch.empty_like(y)
    assert fp8.fp8_linear_forward(x, codes, scale, bias, out=out) is out and torch.equal(out, y)
    odd = torch.empty(12 * 96 + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(12, 96).copy_(x)  # 2 bytes off
    assert torch.equal(fp8.fp8_linear_forward(odd, codes, scale, bias), y)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        other = fp8.fp8_linear_forward(x, codes, scale, bias)
    stream.synchronize()
    assert torch.equal(other, y)
    assert fp8.fp8_linear_forward(x[:0], codes, scale, bias).shape == (0, 80)
    empty = torch.empty(80, 0, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
    none = fp8.fp8_linear_forward(x[:, :0], empty, torch.empty(1, 0, device=cuda_device), bias)
    assert torch.equal(none, bias.expand(12, 80))


def test_input_gradient_against_differences(cuda_device):
    """The forward as a map of the quantised rows is linear: its gradient is the transposed product."""
    x, codes, scale, _, grad = _problem(6, 140, 150, torch.float32, cuda_device)
    x = _quantized_rows(x).float().requires_grad_()
    back = torch.autograd.grad(fp8.fp8_linear(x, codes, scale), x, grad)[0]
    ones = torch.zeros_like(x)
    for column in range(0, 140, 9):
        ones.zero_()[:, column] = 1.0  # quantised exactly: a power of two
        slope = fp8.fp8_linear_forward(ones, codes, scale)  # d y / d x[:, column]
        want = (slope.double() * grad.double()).sum(1)
        # the gradient's own rows are quantised to 4 significant bits: half a step of 2^-3, or the
        # least step 2^-9 of a scale of at most amax / 224
        size = (slope.double().abs() * (grad.double().abs() * 2.0 ** -4 + grad.double().abs().amax(1, keepdim=True)
                                        * 2.0 ** -10 / 224.0)).sum(1)
        assert bool(((back[:, column].double() - want).abs() <= size * 1.001).all())


def test_module_in_a_model_and_under_lora(cuda_device):
    torch.manual_seed(0)
    model = nn.Sequential(nn.Linear(100, 260), nn.GELU(), nn.Linear(260, 64, bias=False)).to(cuda_device, torch.bfloat16)
    dense = [layer.weight.detach().double() for layer in (model[0], model[2])]
    model.requires_grad_(False)
    model[2] = LoRALinear(model[2], 4, 4.0).to(cuda_device)
    assert fp8.quantize_frozen_linears_fp8(model) == ["0", "2.base"]
    x = torch.randn(50, 100, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    y = model(x)
    y.float().square().sum().backward()
    assert y.shape == (50, 64) and x.grad.isfinite().all() and model[2].lora_B.grad.abs().sum() > 0
    for layer, weight in zip((model[0], model[2].base), dense):
        assert float((layer.weight.double() - weight).norm() / weight.norm()) < 0.04  # 4 significant bits
    state = {name: tensor.clone() for name, tensor in model.state_dict().items()}
    assert state["0.weight_fp8"].dtype == torch.float8_e4m3fn
    model.load_state_dict(state)
    model.to(torch.float16)
    assert model[0].weight_scale.dtype == torch.float32 and model[0].weight_fp8.dtype == torch.float8_e4m3fn
    assert model[0](x.detach().half()).dtype == torch.float16
    again = fp8.FrozenFp8Linear.from_codes(state["0.weight_fp8"].contiguous(), state["0.weight_scale"], state["0.bias"])
    assert torch.equal(again(x.detach()), fp8.fp8_linear_forward(x.detach(), model[0].weight_fp8, state["0.weight_scale"],
                                                                 state["0.bias"]))


def test_refusals(cuda_device):
    x, codes, scale, bias, _ = _problem(4, 96, 80, torch.bfloat16, cuda_device)
    unaligned = torch.empty(80, 97, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)[:, :96]
    for arguments in (
        (x[:, :90], codes, scale), (x, codes, scale[:0]), (x, codes, scale.double()), (x, codes.float(), scale),
        (x, codes.cpu(), scale), (x, unaligned, scale), (x.long(), codes, scale), (x, codes, scale, bias[:3]),
        (x, codes, scale, bias.cpu()), (x, codes, scale, bias, torch.int32),
    ):
        with pytest.raises(ValueError):
            fp8.fp8_linear_forward(*arguments)
    with pytest.raises(ValueError):
        fp8.fp8_linear_backward(x, codes, scale)
    with pytest.raises(ValueError):
        fp8.fp8_linear_forward(x, codes, scale, out=torch.empty(4, 80, device=cuda_device))
    with pytest.raises(RuntimeError, match="CUDA"):
        fp8.fp8_linear_forward(x.cpu(), codes, scale)
    with pytest.raises(ValueError, match="Freeze"):
        fp8.FrozenFp8Linear(nn.Linear(4, 4).to(cuda_device))
    with pytest.raises(ValueError):
        fp8.FrozenFp8Linear.from_codes(codes, scale[:0])


@pytest.mark.parametrize("m", [15, 31, 32, 33, 63])
@pytest.mark.parametrize("k,n", [(2048, 1536), (1031, 645)])
def test_few_rows_on_either_side_of_the_kernels(cuda_device, m, k, n):
    """Row counts around the few-row kernel's tiles, reductions long enough to be split and their gradients."""
    x, codes, scale, bias, grad = _problem(m, k, n, torch.float32, cuda_device, seed=2)
    weight = _decoded(codes, scale)
    _check(fp8.fp8_linear_forward(x, codes, scale, bias), _quantized_rows(x), weight.t(), bias)
    _check(fp8.fp8_linear_backward(grad, codes, scale), _quantized_rows(grad), weight)


def test_calls_replay_from_a_graph(cuda_device):
    problems = [_problem(m, 640, 520, torch.bfloat16, cuda_device, seed=4) for m in (3, 150, 2100)]
    want = [fp8.fp8_linear_forward(x, codes, scale, bias) for x, codes, scale, bias, _ in problems]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [fp8.fp8_linear_forward(x, codes, scale, bias) for x, codes, scale, bias, _ in problems]
    for x, *_ in problems:
        x.neg_()
    graph.replay()
    for (x, codes, scale, bias, _), y, before in zip(problems, got, want):
        assert torch.equal(y, fp8.fp8_linear_forward(x, codes, scale, bias)) and not torch.equal(y, before)


def test_offsets_past_32_bits(cuda_device):
    m, k, n = 140_000, 128, 16_384  # 2.3e9 outputs
    x, codes, scale, _, _ = _problem(3, k, n, torch.bfloat16, cuda_device, seed=6)
    rows = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda_device)
    rows[-3:] = x
    y = fp8.fp8_linear_forward(rows, codes, scale)
    _check(y[-3:], _quantized_rows(x), _decoded(codes, scale).t())
    assert not y[: m // 2].any()
    back = fp8.fp8_linear_backward(y, codes, scale)  # reads past 2^31 values
    _check(back[-3:], _quantized_rows(y[-3:]), _decoded(codes, scale))


def test_a_second_gradient_is_refused(cuda_device):
    x, codes, scale, _, grad = _problem(4, 128, 128, torch.float32, cuda_device)
    x.requires_grad_()
    first, = torch.autograd.grad(fp8.fp8_linear(x, codes, scale), x, grad.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(2500, 256, 2052), (2500, 256, 2049), (700, 300, 646), (130, 128, 36)])
def test_tile_outputs_of_any_width_and_alignment_stay_in_their_place(cuda_device, dtype, m, k, n, offset):
    x, codes, scale, bias, grad = _problem(m, k, n, dtype, cuda_device, seed=5)
    weight = _decoded(codes, scale)
    for rows, width, run, want in (
            (x, n, lambda o: fp8.fp8_linear_forward(x, codes, scale, bias, out=o), (weight.t(), bias)),
            (grad, k, lambda o: fp8.fp8_linear_backward(grad, codes, scale, out=o), (weight, None))):
        room = torch.full((m * width + 64,), 7.0, dtype=dtype, device=cuda_device)
        out = room[16 + offset:16 + offset + m * width].view(m, width)
        assert run(out) is out
        _check(out, _quantized_rows(rows), *want)
        assert (room[:16 + offset] == 7.0).all() and (room[16 + offset + m * width:] == 7.0).all()


def test_forward_mode_is_refused(cuda_device):
    from torch.autograd import forward_ad

    x, codes, scale, bias, _ = _problem(4, 96, 80, torch.float32, cuda_device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            fp8.fp8_linear(dual, codes, scale, bias)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            fp8.fp8_linear(dual, codes, scale, bias)
        assert torch.equal(fp8.fp8_linear(x, codes, scale, bias), fp8.fp8_linear_forward(x, codes, scale, bias))
        tracked, y = x.clone().requires_grad_(), fp8.fp8_linear_forward(x, codes, scale)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(fp8.fp8_linear(tracked, codes, scale), tracked, forward_ad.make_dual(y, y))
