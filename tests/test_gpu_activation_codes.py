"""Coded activations on the GPU: codes and decoded values bit for bit against the rule in float64, weight
gradients against float64 products of the decoded values.

Bounds of a gradient: its terms are exact products of 16-bit values; the tensor cores add them 16 at a time to f32
sums, each addition off by at most 2^-22 of the sum of magnitudes (twice a step, for truncating
adders), and splits and warps add a few more; then one rounding to the result's type, half a step.
"""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from moss_image_b200.activation_codes import (CodedActivation, coded_checkpoints, coded_linear, coded_weight_gradient,
                                              decode_activation, encode_activation)
from moss_image_b200.activation_offload import activation_cpu_offload
from moss_image_b200.lora import LoRALinear
from moss_image_b200.quantization import FrozenInt8Linear

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def _rule(x: torch.Tensor):
    """(codes, exponent bytes) of a matrix, in float64 on the CPU."""
    rows, columns = x.shape
    value = x.detach().cpu().double()
    blocks = torch.nn.functional.pad(value, (0, -columns % 32)).view(rows, -1, 32)
    finite = blocks.isfinite().all(-1)
    top = torch.where(finite, blocks.abs().amax(-1), torch.zeros(()).double())
    power = torch.full(top.shape, -126, dtype=torch.int64)
    cap = 9 if x.dtype == F16 else 121
    for p in range(-126, cap):  # raised as long as the block does not fit
        power += (power == p) & (top > 127 * 2.0 ** p)
    codes = (blocks / torch.exp2(power.double())[..., None]).nan_to_num(0, 0, 0).round().clamp(-127, 127)
    codes = torch.where(finite[..., None], codes, 0.0)
    exponents = torch.where(finite, power + 127, 255)
    return codes.view(rows, -1)[:, :columns].to(torch.int8), exponents.to(torch.uint8)


def _values(coded: CodedActivation) -> torch.Tensor:
    power = (coded.exponents.double() - 127).repeat_interleave(32, 1)[:, : coded.codes.shape[1]]
    return coded.codes.double() * torch.exp2(power)


def _tokens(rows, columns, dtype, seed, spread=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, columns, generator=gen, device="cuda")
    return (x * torch.exp(spread * torch.randn(rows, 1, generator=gen, device="cuda"))).to(dtype)


def _same(x):
    coded = encode_activation(x)
    codes, exponents = _rule(x)
    assert torch.equal(coded.codes.cpu(), codes) and torch.equal(coded.exponents.cpu(), exponents)
    decoded = decode_activation(coded)
    assert decoded.dtype == x.dtype and decoded.shape == x.shape
    good = (coded.exponents != 255).repeat_interleave(32, 1)[:, : x.shape[1]]
    assert torch.equal(decoded.double()[good], _values(coded)[good]) and decoded[~good].isnan().all()
    return coded, decoded


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 16), (5, 31), (7, 32), (9, 48), (2, 33), (66, 80), (130, 272), (17, 1090),
                                          (40, 3072), (1, 20000)])
def test_codes_and_decoded_values(cuda_device, rows, columns, dtype):
    x = _tokens(rows, columns, dtype, rows + columns)
    coded, decoded = _same(x)
    top = torch.nn.functional.pad(x.double(), (0, -columns % 32)).view(rows, -1, 32).abs().amax(-1)
    allowed = top.repeat_interleave(32, 1)[:, :columns] / 127
    assert ((decoded.double() - x.double()).abs() <= allowed).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("columns", [64, 45])
def test_ties_extremes_and_empty_blocks(cuda_device, dtype, columns):
    info = torch.finfo(dtype)
    x = torch.zeros(12, columns, device="cuda", dtype=dtype)
    x[1, 0] = info.max
    x[2, 0] = -info.max
    x[3, :] = info.smallest_normal
    x[4, :] = info.smallest_normal * info.eps  # the least value there is
    x[5, 0], x[5, 1:33] = 127.0, torch.arange(32, device="cuda", dtype=dtype) + 0.5  # halves go to the even code
    x[6, 0], x[7, 0] = 127.0 * 4, 127.0 * 4 * (1 + info.eps)  # the last value of a power, and the first past it
    x[8, :] = -info.max
    x[9, 1:20] = -info.max / 3
    x[10, 32:] = 1.0
    _same(x)


@pytest.mark.parametrize("columns", [64, 45])
def test_non_finite_blocks_decode_to_nan(cuda_device, columns):
    x = _tokens(6, columns, BF16, 3)
    x[1, 5], x[2, 40], x[3, 0], x[3, 1] = float("nan"), float("inf"), -float("inf"), float("nan")
    _same(x)


def test_shapes_strides_and_alignment(cuda_device):
    x = torch.randn(4, 6, 3, 96, device="cuda").to(BF16)
    coded = encode_activation(x[:, :, 1])
    assert coded.shape == (4, 6, 96) and torch.equal(decode_activation(coded).flatten(0, 1),
                                                     _same(x[:, :, 1].reshape(24, 96))[1])
    flat = torch.randn(1 + 8 * 64, device="cuda").to(F16)
    _same(flat[1:].view(8, 64))  # rows off the 32-byte grid
    vector = torch.randn(70, device="cuda")
    assert decode_activation(encode_activation(vector)).shape == (70,)
    empty = encode_activation(torch.empty(0, 40, device="cuda", dtype=BF16))
    assert decode_activation(empty).shape == (0, 40)
    assert decode_activation(encode_activation(torch.empty(3, 0, device="cuda", dtype=BF16))).shape == (3, 0)
    half = decode_activation(encode_activation(x[0, 0].to(F32)), BF16)
    assert half.dtype == BF16


def _gradient_bound(dy, values, dtype):
    terms = dy.double().abs().t() @ values.abs()
    exact = dy.double().t() @ values
    slack = (dy.shape[0] / 16 + 64) * 2.0 ** -22 * terms
    return exact, slack + HALF_STEP[dtype] * (exact.abs() + slack) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _assert_gradient(dy, coded, out_dtype=None):
    got = coded_weight_gradient(dy, coded.codes, coded.exponents, out_dtype)
    exact, allowed = _gradient_bound(dy.reshape(-1, dy.shape[-1]), _values(coded), got.dtype)
    worst = ((got.double() - exact).abs() / allowed).max().item()
    assert worst <= 1.0, worst
    return got


GRADIENTS = [  # rows, features, columns: few features; single tiles, split and whole; pair tiles; odd ones of each
    (1, 1, 1), (5, 3, 40), (16, 16, 128), (17, 17, 129), (130, 32, 272), (1500, 32, 96), (4111, 24, 1090), (2300, 5, 3072),
    (1, 33, 16), (127, 40, 48), (128, 128, 128), (129, 136, 200), (1003, 130, 75), (6000, 64, 320), (300, 513, 1090),
    (384, 2304, 2560), (257, 3000, 2501),
]


@pytest.mark.parametrize("rows,features,columns", GRADIENTS)
@pytest.mark.parametrize("dtype,out_dtype", [(BF16, None), (F16, None), (BF16, F32)])
def test_weight_gradient(cuda_device, rows, features, columns, dtype, out_dtype):
    coded = encode_activation(_tokens(rows, columns, dtype, rows, 0.5))
    dy = _tokens(rows, features, dtype, features, 0.5)
    _assert_gradient(dy, coded, out_dtype)


@pytest.mark.parametrize("features", [7, 40])
def test_small_scales_of_f16(cuda_device, features):
    x = _tokens(96, 80, F16, 1, 0.5) * 2.0 ** -12  # powers of two below f16's own
    x[::3] *= 2.0 ** -9
    dy = _tokens(96, features, F16, 2, 0.5)
    _assert_gradient(dy, encode_activation(x))


@pytest.mark.parametrize("features", [8, 64])
def test_non_finite_inputs_reach_the_gradient(cuda_device, features):
    x = _tokens(50, 96, BF16, 1)
    x[7, 40] = float("inf")  # the block of columns 32 to 63 is NaN
    dy = _tokens(50, features, BF16, 2)
    coded = encode_activation(x)
    got = coded_weight_gradient(dy, coded.codes, coded.exponents)
    assert got[:, 32:64].isnan().all() and got[:, :32].isfinite().all() and got[:, 64:].isfinite().all()


def test_gradient_layouts(cuda_device):
    coded = encode_activation(_tokens(300, 100, BF16, 1))
    plain = _tokens(300, 2 * 72, BF16, 2)
    full = _assert_gradient(plain[:, :72].contiguous(), coded)
    assert torch.equal(coded_weight_gradient(plain[:, :72], coded.codes, coded.exponents), full)  # strided
    shifted = torch.empty(1 + 300 * 72, dtype=BF16, device="cuda")[1:].view(300, 72).copy_(plain[:, :72])
    assert torch.equal(coded_weight_gradient(shifted, coded.codes, coded.exponents), full)  # off the 16-byte grid
    assert torch.equal(coded_weight_gradient(plain[:, :72].reshape(3, 100, 72), coded.codes, coded.exponents), full)
    dense = coded.codes.contiguous()  # rows 100 bytes apart: laid out again
    assert torch.equal(coded_weight_gradient(plain[:, :72], dense, coded.exponents), full)
    wide = torch.zeros(300, 160, dtype=torch.int8, device="cuda")[:, :100].copy_(coded.codes)
    assert torch.equal(coded_weight_gradient(plain[:, :72], wide, coded.exponents), full)
    none = coded_weight_gradient(plain[:0, :72], coded.codes[:0], coded.exponents[:0])
    assert none.shape == (72, 100) and not none.any()
    assert coded_weight_gradient(plain[:, :0], coded.codes, coded.exponents).shape == (0, 100)


def test_same_bits_on_a_side_stream_and_in_graphs(cuda_device):
    x, dy = _tokens(3000, 320, BF16, 1), _tokens(3000, 48, BF16, 2)
    thin = dy[:, :24].contiguous()

    def step():
        coded = encode_activation(x)
        return [decode_activation(coded), coded_weight_gradient(dy, coded.codes, coded.exponents),
                coded_weight_gradient(thin, coded.codes, coded.exponents)]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:  # two graphs, each with workspaces of its own
        with torch.cuda.graph(graph):
            outs.append(step())
    x.mul_(-1)
    for graph in graphs:
        graph.replay()
    for captured in outs:
        assert torch.equal(captured[0], -first[0])
        assert all(torch.equal(a, -b) for a, b in zip(captured[1:], first[1:]))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("with_bias", [True, False])
def test_coded_linear(cuda_device, dtype, with_bias):
    x = _tokens(2 * 60, 96, dtype, 1, 0.3).view(2, 60, 96).requires_grad_()
    weight = (0.1 * _tokens(40, 96, dtype, 2, 0.1)).requires_grad_()
    bias = _tokens(1, 40, dtype, 3, 0.1)[0].requires_grad_() if with_bias else None
    leaves = [x, weight] + ([bias] if with_bias else [])
    dy = _tokens(120, 40, dtype, 4, 0.1).view(2, 60, 40)
    y = coded_linear(x, weight, bias)
    plain = torch.nn.functional.linear(x, weight, bias)
    assert torch.equal(y, plain)
    got, kept = torch.autograd.grad(y, leaves, dy), torch.autograd.grad(plain, leaves, dy)
    assert torch.equal(got[0], kept[0])
    coded = encode_activation(x)
    assert torch.equal(got[1], coded_weight_gradient(dy, coded.codes, coded.exponents))
    # the codes are off by a 254th of their block's largest magnitude on average less: a percent of the gradient
    assert (got[1].float() - kept[1].float()).norm() <= 0.02 * kept[1].float().norm()
    if with_bias:
        exact = dy.double().sum((0, 1))
        assert ((got[2].double() - exact).abs() <= 120 * 2.0 ** -24 * dy.double().abs().sum((0, 1))
                + HALF_STEP[dtype] * exact.abs()).all()
    shared = torch.autograd.grad(coded_linear(x, weight, bias, coded=coded), weight, dy)[0]
    assert torch.equal(shared, got[1])
    frozen = coded_linear(x, weight.detach())
    assert torch.equal(torch.autograd.grad(frozen, x, dy)[0], got[0])
    with torch.no_grad():
        assert not coded_linear(x, weight, bias).requires_grad


def test_coded_linear_keeps_codes_only(cuda_device):
    x = torch.randn(4096, 1024, device="cuda", dtype=BF16)
    weight = torch.randn(64, 1024, device="cuda", dtype=BF16, requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = coded_linear(x * 1.0, weight)
    held = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert held <= 1.05 * x.numel()  # 33/32 of a byte a value


def test_coded_checkpoint_recomputes_from_the_decoded_input(cuda_device):
    torch.manual_seed(0)
    block = torch.nn.Sequential(torch.nn.Linear(64, 64), torch.nn.GELU(), torch.nn.Linear(64, 64)).to("cuda", BF16)
    leaf = torch.randn(2, 50, 64, device="cuda").to(BF16).requires_grad_()
    x = leaf * 1.0
    dy = torch.randn(2, 50, 64, device="cuda").to(BF16)
    with coded_checkpoints(x):
        y = checkpoint(block, x, use_reentrant=False)
    assert torch.equal(y, block(x))
    got = torch.autograd.grad(y, [leaf, *block.parameters()], dy)
    near = decode_activation(encode_activation(x)).requires_grad_()
    expected = torch.autograd.grad(block(near), [near, *block.parameters()], dy)
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("width", [64, 50])
def test_codes_leave_with_the_offload(cuda_device, width):
    torch.manual_seed(1)
    block = torch.nn.Linear(width, width).to("cuda", BF16)
    leaf = torch.randn(7, width, device="cuda").to(BF16).requires_grad_()
    dy = torch.randn(7, width, device="cuda").to(BF16)
    grads = []
    for offload in (False, True):
        scope = activation_cpu_offload(block, offload, leaf.device)
        x = leaf * 1.0
        with scope, coded_checkpoints(x, scope):
            y = checkpoint(block, x, use_reentrant=False)
        grads.append(torch.autograd.grad(y, [leaf, *block.parameters()], dy))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_refusals(cuda_device):
    x = torch.randn(8, 64, device="cuda", dtype=BF16)
    coded = encode_activation(x)
    with pytest.raises(ValueError, match="float16"):
        encode_activation(x.double())
    with pytest.raises(ValueError, match="16 or bfloat16"):
        coded_weight_gradient(x.float(), coded.codes, coded.exponents)
    with pytest.raises(ValueError, match="one row"):
        coded_weight_gradient(x[:7], coded.codes, coded.exponents)
    with pytest.raises(ValueError, match="exponents"):
        coded_weight_gradient(x, coded.codes, coded.exponents[:, :1])
    with pytest.raises(ValueError, match="int8"):
        coded_weight_gradient(x, coded.codes.view(torch.uint8), coded.exponents)
    with pytest.raises(ValueError, match="device"):
        coded_weight_gradient(x, coded.codes.cpu(), coded.exponents.cpu())
    with pytest.raises(ValueError, match="one dtype"):
        coded_linear(x, torch.randn(4, 64, device="cuda"))
    with pytest.raises(ValueError, match="not those"):
        coded_linear(x, torch.randn(4, 64, device="cuda", dtype=BF16), coded=encode_activation(x[:4]))
    with torch.autocast("cuda", F16), pytest.raises(ValueError, match="autocast"):
        coded_linear(x, torch.randn(4, 64, device="cuda", dtype=BF16))
    weight = torch.randn(4, 64, device="cuda", dtype=BF16, requires_grad=True)
    slope, = torch.autograd.grad(coded_linear(x.requires_grad_(), weight).float().square().sum(), weight, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(slope.float().sum(), weight)


@pytest.mark.parametrize("features", [8, 40])
def test_codes_past_float16(cuda_device, features):
    """Codes of wider types under a float16 gradient: refused where the caller says so, else what float16 makes of their values."""
    x = torch.zeros(48, 96, device="cuda")
    x[3, 0], x[3, 5] = 127.0 * 2.0 ** 16, 2.0 ** 16  # past float16; the block's other values are zeros
    x[4, 40], x[4, 41] = 127.0 * 2.0 ** 40, 1.0
    x[5, 64:] = 60000.0  # a block of float16 values whose power of two is one
    x[6, :32] = 2.0 ** -30
    x[7, 70] = float("nan")
    coded = encode_activation(x)
    dy = torch.randn(48, features, device="cuda").to(F16)
    with pytest.raises(ValueError, match="does not hold"):
        coded_weight_gradient(dy, coded.codes, coded.exponents, coded_dtype=F32)
    got = coded_weight_gradient(dy, coded.codes, coded.exponents, F32)
    exact = dy.double().t() @ decode_activation(coded, F16).double()
    assert torch.equal(got.isnan(), exact.isnan()) and torch.equal(got.isinf(), exact.isinf())
    good = exact.isfinite()
    assert ((got.double() - exact).abs()[good] <= 2.0 ** -20 * (dy.double().abs().t() @ x.abs().nan_to_num(0).double())[good]).all()
    wide = coded_weight_gradient(dy.to(BF16), coded.codes, coded.exponents, F32, coded_dtype=F32)
    assert torch.equal(wide.isfinite(), torch.arange(96, device="cuda").lt(64).expand_as(wide))


def test_codes_of_another_dtype_are_refused(cuda_device):
    x = torch.randn(8, 64, device="cuda", dtype=F16)
    weight = torch.randn(4, 64, device="cuda", dtype=F16, requires_grad=True)
    with pytest.raises(ValueError, match="another dtype"):
        coded_linear(x, weight, coded=encode_activation(x.to(BF16)))
    base = torch.nn.Linear(64, 32).to("cuda", F16).requires_grad_(False)
    layer = LoRALinear(FrozenInt8Linear(base), 4, 8.0).to("cuda")
    torch.nn.init.normal_(layer.lora_B, std=0.05)
    with pytest.raises(ValueError, match="another dtype"):
        layer(x, encode_activation(x.to(BF16)))
    # float16 adapters of wider tokens keep the tokens
    tokens = torch.randn(8, 64, device="cuda", dtype=BF16)
    grads = []
    for codes in (None, encode_activation(tokens)):
        with torch.autocast("cuda", F16):
            y = layer(tokens, codes)
        grads.append(torch.autograd.grad(y.float().sum(), layer.lora_A)[0])
    assert torch.equal(*grads)


def test_only_the_tokens_of_a_checkpoint_are_coded(cuda_device):
    """Another input of the tokens' shape and dtype (a context) stays whole."""
    torch.manual_seed(2)
    weight = torch.randn(64, 64, device="cuda", dtype=BF16, requires_grad=True)

    def block(x, context):
        return (x @ weight) * context

    leaf, context = (torch.randn(2, 50, 64, device="cuda").to(BF16) for _ in range(2))
    x, other = leaf.requires_grad_() * 1.0, context.requires_grad_() * 1.0
    dy = torch.randn(2, 50, 64, device="cuda").to(BF16)
    with coded_checkpoints(x):
        y = checkpoint(block, x, other, use_reentrant=False)
    got = torch.autograd.grad(y, [leaf, context, weight], dy)
    near = decode_activation(encode_activation(x)).requires_grad_()
    expected = torch.autograd.grad(block(near, context), [near, context, weight], dy)
    assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("features,copied", [(64, False), (24, False), (60, True)])
def test_room_for_a_copy_of_the_gradient_only_where_one_is_made(cuda_device, features, copied):
    rows, columns = 40000, 64
    coded = encode_activation(_tokens(rows, columns, BF16, 1, 0.5))
    dy = _tokens(rows, features, BF16, 2, 0.5)
    coded_weight_gradient(dy, coded.codes, coded.exponents)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    coded_weight_gradient(dy, coded.codes, coded.exponents)
    used = torch.cuda.memory_stats()["requested_bytes.all.peak"] - before
    decoded = rows * columns * 2 if features > 32 else 0
    partials = 4 * 160 * 128 * 128  # one tile of sums for each multiprocessor, at most
    padded = rows * 64 * 2 if copied else 0
    assert decoded + padded <= used <= decoded + padded + partials
    nothing = encode_activation(torch.empty(40, 0, device="cuda", dtype=BF16))
    assert coded_weight_gradient(dy[:40], nothing.codes, nothing.exponents).shape == (features, 0)


def test_second_derivatives_are_refused(cuda_device):
    coded = encode_activation(torch.randn(40, 64, device="cuda", dtype=BF16))
    dy = torch.randn(40, 48, device="cuda", dtype=BF16, requires_grad=True)
    got = coded_weight_gradient(dy * 1.0, coded.codes, coded.exponents, F32)
    assert torch.equal(got, coded_weight_gradient(dy.detach(), coded.codes, coded.exponents, F32))
    with pytest.raises(NotImplementedError, match="no gradient"):
        got.sum().backward()
    # an adapter on codes, whose own backward pass records its steps
    base = torch.nn.Linear(64, 32).to("cuda", BF16).requires_grad_(False)
    layer = LoRALinear(FrozenInt8Linear(base), 4, 8.0).to("cuda")
    torch.nn.init.normal_(layer.lora_B, std=0.05)
    x = torch.randn(8, 64, device="cuda", dtype=BF16)
    with torch.autocast("cuda", BF16):
        y = layer(x, encode_activation(x))
    slope, = torch.autograd.grad(y.float().square().sum(), layer.lora_A, create_graph=True)
    with pytest.raises(NotImplementedError, match="no gradient"):
        torch.autograd.grad(slope.square().sum(), layer.lora_B)


@pytest.mark.parametrize("rows,features,columns", [((2, 5), 0, 32), ((0,), 24, 32), ((3,), 24, 0), ((), 24, 32)])
def test_coded_linear_of_nothing(cuda_device, rows, features, columns):
    x = torch.randn(*rows, columns, device="cuda").to(BF16).requires_grad_()
    weight, bias = (torch.randn(*shape, device="cuda").to(BF16).requires_grad_() for shape in ((features, columns), (features,)))
    y, plain = coded_linear(x, weight, bias), torch.nn.functional.linear(x, weight, bias)
    dy = torch.randn_like(plain)
    got, whole = (torch.autograd.grad(t, [x, weight, bias], dy) for t in (y, plain))
    assert torch.equal(y, plain) and all(a.shape == b.shape for a, b in zip(got, whole))
    assert torch.equal(got[0], whole[0]) and torch.equal(got[2], whole[2])
