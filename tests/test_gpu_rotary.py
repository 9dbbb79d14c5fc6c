"""Rotary positions on the GPU against the same turn in float64."""

from __future__ import annotations

import pytest
import torch

from moss_image_b200.rotary import apply_rotary, rotary_frequencies, rotary_table

pytestmark = pytest.mark.gpu

# one rounding to the type (unit roundoff) and, for float16, half a subnormal step
ROUNDING = {torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.float32: (2.0 ** -24, 0.0)}


def _turn(x, cos, sin, interleaved, sign=1.0):
    """The turn in float64; cos and sin are [tokens, half] or [batch, tokens, half]."""
    half = cos.shape[-1]
    v, out = x.double(), x.double().clone()
    c, s = cos.double().unsqueeze(-2), sign * sin.double().unsqueeze(-2)
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = v[..., first], v[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    return out


def _check(got, want, x):
    relative, absolute = ROUNDING[x.dtype]
    # two products and a sum in f32 before that rounding: 3 roundings of at most |x| sqrt(2) each
    room = relative * want.abs() + absolute + 3 * 1.5 * 2.0 ** -24 * x.double().abs().amax(-1, keepdim=True)
    assert bool(((got.double() - want).abs() <= room).all())


def _table(rows, half, device):
    cos, sin = rotary_table(torch.arange(rows, device=device), rotary_frequencies(2 * half, device=device)) if half else (
        torch.zeros(rows, 0, device=device),) * 2
    return cos, sin


@pytest.mark.parametrize("dtype", list(ROUNDING))
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("batch,tokens,q_heads,k_heads,dim,rotary", [
    (1, 1, 1, 1, 2, 2), (2, 7, 3, 1, 128, 128), (1, 130, 24, 8, 128, 64), (3, 5, 5, 2, 80, 40), (1, 33, 9, 9, 96, 80),
    (2, 17, 2, 2, 7, 6), (1, 9, 4, 4, 64, 0), (1, 600, 6, 1, 256, 256), (1, 4, 4, 3, 20, 12),
])
def test_forward_and_gradient(cuda_device, dtype, interleaved, batch, tokens, q_heads, k_heads, dim, rotary):
    gen = torch.Generator().manual_seed(tokens * dim + q_heads)
    q = torch.randn(batch, tokens, q_heads, dim, generator=gen).to(cuda_device, dtype).requires_grad_()
    k = torch.randn(batch, tokens, k_heads, dim, generator=gen).to(cuda_device, dtype).requires_grad_()
    cos, sin = _table(tokens, rotary // 2, cuda_device)
    out = apply_rotary(q, k, cos, sin, interleaved=interleaved)
    grads = [torch.randn(t.shape, generator=gen).to(cuda_device, dtype) for t in (q, k)]
    back = torch.autograd.grad(out, (q, k), grads)
    for x, y, g, dx in zip((q, k), out, grads, back):
        assert y.dtype == dtype and y.shape == x.shape
        _check(y.detach(), _turn(x.detach(), cos, sin, interleaved), x.detach())
        _check(dx, _turn(g, cos, sin, interleaved, -1.0), g)


@pytest.mark.parametrize("interleaved", [True, False])
def test_views_of_a_fused_projection_and_positions(cuda_device, interleaved):
    gen = torch.Generator().manual_seed(3)
    fused = torch.randn(2, 37, (6 + 2 + 2) * 64, generator=gen).to(cuda_device, torch.bfloat16)
    q, k = fused[..., : 6 * 64].unflatten(-1, (6, 64)), fused[..., 6 * 64 : 8 * 64].unflatten(-1, (2, 64))
    cos, sin = _table(500, 32, cuda_device)
    for places in (torch.randint(0, 500, (2, 37), generator=gen), torch.randint(0, 500, (37,), generator=gen)):
        places = places.to(cuda_device)
        out = apply_rotary(q, k, cos, sin, interleaved=interleaved, positions=places)
        for x, y in zip((q, k), out):
            _check(y, _turn(x, cos[places], sin[places], interleaved), x)


def test_packed_heads_first_and_unaligned_views(cuda_device):
    gen = torch.Generator().manual_seed(5)
    cos, sin = _table(19, 16, cuda_device)
    heads_first = torch.randn(4, 19, 32, generator=gen).to(cuda_device, torch.float16).transpose(0, 1)
    store = torch.randn(19 * 2 * 33 + 1, generator=gen).to(cuda_device, torch.float16)
    odd = store[1:].view(19, 2, 33)[..., :32]  # 2 bytes off any wider boundary, rows 66 bytes apart
    last_strided = torch.randn(19, 32, 3, generator=gen).to(cuda_device, torch.float16).transpose(1, 2)
    for k in (odd, last_strided):
        out = apply_rotary(heads_first, k, cos, sin, interleaved=False)
        for x, y in zip((heads_first, k), out):
            _check(y, _turn(x[None], cos, sin, False)[0], x)


def test_gradient_against_differences(cuda_device):
    gen = torch.Generator().manual_seed(6)
    q = torch.randn(1, 5, 2, 16, generator=gen).to(cuda_device).requires_grad_()
    k = torch.randn(1, 5, 1, 16, generator=gen).to(cuda_device).requires_grad_()
    cos, sin = _table(5, 6, cuda_device)
    weights = [torch.randn(t.shape, generator=gen).to(cuda_device) for t in (q, k)]

    def loss(a, b):
        return sum((y.double() * w.double()).sum() for y, w in zip(apply_rotary(a, b, cos, sin), weights))

    back = torch.autograd.grad(loss(q, k), (q, k))
    with torch.no_grad():
        for which, (x, g) in enumerate(zip((q, k), back)):
            for index in range(0, x.numel(), 7):
                step = torch.zeros_like(x)
                step.view(-1)[index] = 0.5
                pair = [loss(*(t + sign * step if i == which else t for i, t in enumerate((q, k)))) for sign in (1, -1)]
                # the map is linear: differences are exact up to the f32 roundings of about 2^-22 in either loss
                assert abs(float(pair[0] - pair[1]) - float(g.view(-1)[index])) < 2.0 ** -18


def test_positions_outside_the_table_read_nan_and_leave_the_rest(cuda_device):
    cos, sin = _table(8, 4, cuda_device)
    q = torch.ones(1, 4, 2, 8, device=cuda_device)
    places = torch.tensor([7, 8, -1, 0], device=cuda_device)
    out, _ = apply_rotary(q, q, cos, sin, positions=places)
    assert out[0, 1:3].isnan().all() and out[0, 0].isfinite().all() and out[0, 3].isfinite().all()


def test_empty_inputs_and_another_stream(cuda_device):
    cos, sin = _table(4, 4, cuda_device)
    q = torch.zeros(0, 4, 2, 8, device=cuda_device)
    assert apply_rotary(q, q, cos, sin)[0].shape == q.shape
    q = torch.zeros(1, 0, 2, 8, device=cuda_device)
    assert apply_rotary(q, q, cos, sin)[1].shape == q.shape
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        x = torch.randn(1, 4, 2, 8, device=cuda_device)
        y, _ = apply_rotary(x, x, cos, sin)
    stream.synchronize()
    _check(y, _turn(x, cos, sin, True), x)


def test_refusals(cuda_device):
    q = torch.zeros(1, 4, 2, 8, device=cuda_device)
    cos, sin = _table(4, 4, cuda_device)
    places = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    for bad in (
        dict(k=q.cpu()), dict(k=q.half()), dict(k=q[:, :3]), dict(k=q[..., :6]), dict(k=q[0]), dict(cos=cos.half()),
        dict(cos=cos[:3], sin=sin[:3]), dict(cos=cos[:, :3]), dict(cos=torch.zeros(4, 5, device=cuda_device),
                                                                   sin=torch.zeros(4, 5, device=cuda_device)),
        dict(sin=sin.cpu()), dict(positions=places.int()), dict(positions=places[:3]), dict(positions=places.cpu()),
        dict(positions=places.view(4, 1)), dict(q=q.long(), k=q.long()), dict(q=q[0, 0], k=q[0, 0]),
    ):
        arguments = {**dict(q=q, k=q, cos=cos, sin=sin, positions=None), **bad}
        with pytest.raises(ValueError):
            apply_rotary(arguments["q"], arguments["k"], arguments["cos"], arguments["sin"],
                         positions=arguments["positions"])


def test_second_gradient(cuda_device):
    """The turn is linear, so the gradient's own gradient is the turn again."""
    gen = torch.Generator().manual_seed(8)
    q = torch.randn(1, 6, 2, 16, generator=gen).to(cuda_device).requires_grad_()
    cos, sin = _table(6, 8, cuda_device)
    weight = torch.randn(1, 6, 2, 16, generator=gen).to(cuda_device).requires_grad_()
    grad, = torch.autograd.grad(apply_rotary(q, q, cos, sin)[0], q, weight, create_graph=True)
    direction = torch.randn(1, 6, 2, 16, generator=gen).to(cuda_device)
    again, = torch.autograd.grad(grad, weight, direction)
    _check(again, _turn(direction, cos, sin, True), direction)


def test_offsets_past_32_bits(cuda_device):
    tokens, heads, dim = 140_000, 64, 256  # 2.3e9 values
    q = torch.zeros(1, tokens, heads, dim, dtype=torch.bfloat16, device=cuda_device)
    tail = torch.randn(1, 3, heads, dim, generator=torch.Generator().manual_seed(9)).to(cuda_device, torch.bfloat16)
    q[:, -3:] = tail
    cos, sin = _table(tokens, dim // 2, cuda_device)
    out, small = apply_rotary(q, q[:, :, :1], cos, sin, interleaved=False)
    _check(out[:, -3:], _turn(tail, cos[-3:], sin[-3:], False), tail)
    assert torch.equal(small[:, -3:], out[:, -3:, :1]) and not out[:, : tokens // 2].any()


def test_forward_mode_is_refused(cuda_device):
    from torch.autograd import forward_ad

    q = torch.randn(1, 4, 2, 8, device=cuda_device)
    cos, sin = _table(4, 4, cuda_device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        tables = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (cos, sin)]
        for arguments in ((dual, q, cos, sin), (q, dual, cos, sin), (q, q, tables[0], sin), (q, q, cos, tables[1]),
                          (dual, q.clone().requires_grad_(), cos, sin)):
            with pytest.raises(NotImplementedError):
                apply_rotary(*arguments)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                apply_rotary(*arguments)
        assert torch.equal(apply_rotary(q, q, cos, sin)[0], apply_rotary(q, q, cos, sin)[1])
        tracked = q.clone().requires_grad_()
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(apply_rotary(tracked, q, cos, sin)[0], tracked, dual)


def test_tables_that_ask_for_a_gradient_are_refused(cuda_device):
    q = torch.randn(1, 4, 2, 8, device=cuda_device)
    cos, sin = _table(4, 4, cuda_device)
    learned = cos.clone().requires_grad_()
    for arguments in ((q, q, learned, sin), (q, q, cos, learned), (q.clone().requires_grad_(), q, learned, sin)):
        with pytest.raises(ValueError, match="gradient"):
            apply_rotary(*arguments)
    with torch.no_grad():
        assert torch.equal(apply_rotary(q, q, learned, sin)[0], apply_rotary(q, q, cos, sin)[0])
