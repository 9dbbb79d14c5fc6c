"""The orthogonalised update on the GPU against the same iteration in float64."""

from __future__ import annotations

import pytest
import torch

from moss_image_b200.muon import COEFFICIENTS, Muon, orthogonalize

pytestmark = pytest.mark.gpu

# The result's rounding to bfloat16 alone is off by 1.66e-3 (relative 2-norm: the root mean square of
# a uniform half-step error over a mantissa uniform in its logarithm). The iteration may add as
# much again in square: 1.5 times the rounding in all.
WITHIN = 1.5 * 1.66e-3


def _exact(update, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    x = update.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp_min(eps)
    for step in range(steps):
        a, b, c = coefficients if not isinstance(coefficients[0], tuple) else coefficients[step]
        gram = x @ x.mT
        x = a * x + (b * gram + c * gram @ gram) @ x
    return x.mT if tall else x


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


def _updates(kind, shape, device, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    *lead, m, n = shape
    base = torch.randn(*shape, generator=gen, device=device)
    if kind == "strong":  # a few directions 80 times stronger than all the others together
        base = base + 30.0 * torch.randn(*lead, m, 8, generator=gen, device=device) @ torch.randn(*lead, 8, n, generator=gen,
                                                                                                   device=device)
    elif kind == "rows":
        base = base * torch.exp(torch.randn(*lead, m, 1, generator=gen, device=device))
    elif kind == "decay":
        base = base * (torch.arange(m, device=device) + 1.0).reciprocal()[:, None]
    return 1e-3 * base


SHAPES = [(16, 16), (1, 40), (40, 1), (3, 5), (17, 300), (32, 3072), (3072, 32), (64, 64), (61, 517), (65, 65), (100, 300),
          (300, 100), (128, 128), (129, 257), (521, 1000), (1000, 521), (384, 2048), (2304, 700)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_one_matrix(cuda_device, shape, dtype):
    update = _updates("plain", shape, cuda_device, seed=shape[0]).to(dtype)
    got = orthogonalize(update)
    assert got.dtype == torch.bfloat16 and got.shape == update.shape
    # few values do not average: one rounding step of each is 2^-8 at most
    assert _off(got, _exact(update)) < (WITHIN if update.numel() >= 4096 else 2.0 ** -8 + 1e-4)


@pytest.mark.parametrize("kind", ["strong", "rows", "decay"])
@pytest.mark.parametrize("shape", [(32, 1024), (256, 256), (640, 1500), (1500, 640), (1024, 1024)])
def test_uneven_spectra_keep_their_precision(cuda_device, shape, kind):
    update = _updates(kind, shape, cuda_device, seed=3)
    assert _off(orthogonalize(update), _exact(update)) < WITHIN


@pytest.mark.parametrize("shape", [(5, 24, 200), (3, 200, 24), (3, 130, 150), (2, 2, 300, 200), (7, 512, 512), (2, 1100, 1300)])
def test_batches_are_their_matrices_one_by_one(cuda_device, shape):
    update = _updates("rows", shape, cuda_device, seed=4)
    got, want = orthogonalize(update), _exact(update)
    for one, exact in zip(got.flatten(0, -3), want.flatten(0, -3)):
        assert _off(one, exact) < WITHIN
    assert torch.equal(got, orthogonalize(update))


@pytest.mark.parametrize("shape", [(24, 100), (200, 300)])
def test_steps_coefficients_and_out(cuda_device, shape):
    update = _updates("plain", shape, cuda_device, seed=5)
    cubic = (1.5, -0.5, 0.0)
    each = ((3.4445, -4.7750, 2.0315), (2.5, -2.0, 0.5), (1.875, -1.25, 0.375))
    for steps, coefficients in ((1, COEFFICIENTS), (2, cubic), (12, cubic), (3, each)):
        assert _off(orthogonalize(update, steps, coefficients), _exact(update, steps, coefficients)) < 2.0 ** -8
    out = torch.empty(shape, dtype=torch.bfloat16, device=cuda_device)
    assert orthogonalize(update, out=out) is out and torch.equal(out, orthogonalize(update))
    # 12 cubic steps converge for singular values that started above 1 / 1.5^11
    converged = orthogonalize(update, 16, cubic).double()
    square = converged @ converged.mT
    assert float((square - torch.eye(shape[0], device=cuda_device)).abs().max()) < 0.02


@pytest.mark.parametrize("shape", [(2, 20, 60), (2, 150, 210)])
def test_zero_tiny_large_and_nonfinite_matrices(cuda_device, shape):
    update = _updates("plain", shape, cuda_device, seed=6)
    clean = orthogonalize(update)
    update[1] = 0.0
    got = orthogonalize(update)
    assert torch.equal(got[0], clean[0]) and not got[1].any()
    update[1] = update[0] * 1e-9  # below eps: scaled by 1 / eps, as the definition says
    assert _off(orthogonalize(update)[1], _exact(update)[1]) < 2.0 ** -8
    update[1] = update[0] * 1e12
    assert _off(orthogonalize(update)[1], _exact(update)[1]) < 2.0 ** -8
    for value in (float("nan"), float("inf")):
        update[1] = update[0]
        update[1, 3, 7] = value
        got = orthogonalize(update)
        assert torch.equal(got[0], clean[0]) and got[1].isnan().all()


def test_strides_streams_and_empty(cuda_device):
    update = _updates("plain", (200, 150), cuda_device, seed=7)
    got = orthogonalize(update)
    assert torch.equal(orthogonalize(update.t().contiguous().t()), got)
    odd = torch.empty(200 * 150 + 1, device=cuda_device)[1:].view(200, 150).copy_(update)
    assert torch.equal(orthogonalize(odd), got)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        other = orthogonalize(update)
    stream.synchronize()
    assert torch.equal(other, got)
    assert orthogonalize(update[:0]).shape == (0, 150) and orthogonalize(update[None, :, :0]).shape == (1, 200, 0)
    assert orthogonalize(update.expand(0, 200, 150)).shape == (0, 200, 150)


def test_optimizer_step_matches_its_formula(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    shapes = [(96, 160), (160, 96), (96, 160), (24, 300)]
    params = [torch.nn.Parameter(torch.randn(*s, generator=gen, device=cuda_device)) for s in shapes]
    mine = [p.detach().double() for p in params]
    buffers = [torch.zeros_like(p) for p in mine]
    optimizer = Muon(params, lr=0.02, momentum=0.9, weight_decay=0.1)
    for _ in range(3):
        for p, w, m in zip(params, mine, buffers):
            p.grad = torch.randn(p.shape, generator=gen, device=cuda_device)
            m.mul_(0.9).add_(p.grad.double())
            direction = _exact(p.grad.double() + 0.9 * m)
            w.mul_(1 - 0.02 * 0.1).sub_(0.02 * 0.2 * max(p.shape) ** 0.5 * direction)
        optimizer.step()
    for p, w in zip(params, mine):
        # three updates, each off by at most WITHIN of its norm 0.004 sqrt(max) sqrt(min) 1.2, and f32 weights
        room = 3 * WITHIN * 0.004 * (p.shape[0] * p.shape[1]) ** 0.5 * 1.2 + 1e-6 * float(w.norm())
        assert float((p.detach().double() - w).norm()) < room


def test_refusals(cuda_device):
    update = torch.zeros(8, 8, device=cuda_device)
    for arguments in (dict(steps=0), dict(steps=17), dict(eps=0.0), dict(eps=float("inf")), dict(coefficients=(1.0, 2.0)),
                      dict(coefficients=((1.0, 0.0, 0.0),) * 2), dict(coefficients=(40.0, 0.0, 0.0)),
                      dict(coefficients=(float("nan"), 0.0, 0.0)), dict(out=update)):
        with pytest.raises(ValueError):
            orthogonalize(update, **arguments)
    with pytest.raises(ValueError):
        orthogonalize(update[0])
    with pytest.raises(ValueError):
        orthogonalize(update.long())
    with pytest.raises(RuntimeError, match="CUDA"):
        orthogonalize(update.cpu())
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(4, device=cuda_device))])
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(update)], momentum=1.0)


def test_calls_replay_from_a_graph(cuda_device):
    updates = [_updates("rows", shape, cuda_device, seed=9) for shape in ((5, 20, 300), (200, 330))]
    for update in updates:
        orthogonalize(update)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [orthogonalize(update) for update in updates]
    for update in updates:
        update.copy_(update.flip(-1))
    graph.replay()
    for update, direction in zip(updates, got):
        assert torch.equal(direction, orthogonalize(update))


def test_offsets_past_32_bits(cuda_device):
    update = torch.zeros(33_000, 64, 1024, dtype=torch.bfloat16, device=cuda_device)  # 2.2e9 values
    update[-1] = _updates("rows", (64, 1024), cuda_device, seed=10).bfloat16()
    direction = orthogonalize(update)
    assert _off(direction[-1], _exact(update[-1])) < WITHIN and not direction[-2].any()
    del direction, update
    wide = torch.zeros(1100, 512, 4096, dtype=torch.bfloat16, device=cuda_device)  # 2.3e9 values, iterated in float16
    wide[-1] = _updates("rows", (512, 4096), cuda_device, seed=11).bfloat16()
    direction = orthogonalize(wide)
    assert _off(direction[-1], _exact(wide[-1])) < WITHIN and not direction[-2].any()


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("shape", [(2, 200, 1501), (2, 200, 1502), (2, 130, 1504), (1, 257, 1000), (2, 301, 290)])
def test_results_of_any_width_and_alignment_stay_in_their_place(cuda_device, shape, offset):
    update = _updates("rows", shape, cuda_device, seed=8)
    room = torch.full((update.numel() + 64,), 7.0, dtype=torch.bfloat16, device=cuda_device)
    out = room[16 + offset:16 + offset + update.numel()].view(shape)
    assert orthogonalize(update, out=out) is out
    assert torch.equal(out, orthogonalize(update)) and _off(out, _exact(update)) < WITHIN
    assert (room[:16 + offset] == 7.0).all() and (room[16 + offset + update.numel():] == 7.0).all()


@pytest.mark.parametrize("scale", [1e-42, 1e-36, 1e-28, 1e-25, 1e-23, 1e-20, 1e25, 3e37])
@pytest.mark.parametrize("shape", [(2, 12, 60), (2, 60, 12), (2, 32, 1100), (2, 1100, 32), (2, 61, 300), (2, 300, 64)])
def test_small_sides_at_the_ends_of_the_range(cuda_device, shape, scale):
    """Squares of these values leave float32; the values and the result do not."""
    update = _updates("rows", shape, cuda_device, seed=12)
    update[1] = update[0] / update[0].abs().amax() * scale
    clean = orthogonalize(update[0])
    for dtype in (torch.float32, torch.bfloat16):
        for eps in (1e-7, 1e-30):
            given = update.to(dtype)
            want = _exact(given, eps=eps)
            got = orthogonalize(given, eps=eps)
            if float(want[1].abs().amax()) < 3e38:  # (below eps, a step only multiplies: tiny over a tiny eps may overflow)
                # (1e-42 is zero in bfloat16)
                assert float((got[1].double() - want[1]).norm()) <= (2.0 ** -8 + 1e-4) * float(want[1].norm())
    assert _off(orthogonalize(update)[0], clean.double()) < 2.0 ** -8


def test_small_sides_with_tiny_and_huge_columns(cuda_device):
    update = _updates("plain", (16, 6000), cuda_device, seed=13)
    update[:, :2500] *= 1e-30
    update[:, 2500:] *= 1e30
    got, want = orthogonalize(update), _exact(update)
    assert _off(got[:, 2500:], want[:, 2500:]) < WITHIN


@pytest.mark.parametrize("shape", [(2, 150, 210), (2, 210, 150)])
@pytest.mark.parametrize("scale,eps", [(1e37, 1e-7), (1e-40, 1e-42)])
def test_large_sides_at_the_ends_of_the_range(cuda_device, shape, scale, eps):
    """Finite values whose norm, or its reciprocal in the iteration's units, leaves float32."""
    update = _updates("plain", shape, cuda_device, seed=14)
    update[1] = update[0] / update[0].abs().amax() * 4.0 * scale
    got, want = orthogonalize(update, eps=eps), _exact(update, eps=eps)
    assert _off(got[1], want[1]) < 2.0 ** -8 and _off(got[0], want[0]) < WITHIN


@pytest.mark.parametrize("shape", [(3, 150, 210), (3, 210, 150), (3, 513, 300)])
@pytest.mark.parametrize("scale", [1e-40, 1e-30, 1e-20, 1e-15, 1e-12])
def test_large_sides_far_below_eps(cuda_device, shape, scale):
    """G / eps is then far below float16's range next to matrices that are not, and so is the result."""
    update = _updates("rows", shape, cuda_device, seed=19)
    update[1] = update[0] / update[0].abs().amax() * scale
    got, want = orthogonalize(update), _exact(update)
    for i, one in enumerate(want):
        assert _off(got[i], one) < WITHIN, (i, scale)
    assert torch.equal(got[0], orthogonalize(update[:1])[0])


@pytest.mark.parametrize("shape", [(256, 400), (400, 256), (2, 130, 700)])
def test_late_steps_that_grow_small_values_keep_their_precision(cuda_device, shape):
    """Later steps that multiply small singular values by 5 each, against the usual 3.4."""
    update = _updates("strong", shape, cuda_device, seed=18)
    growing = ((3.0, -3.0, 1.0), (5.0, -5.0, 1.0), (5.0, -5.0, 1.0))
    assert _off(orthogonalize(update, 3, growing), _exact(update, 3, growing)) < WITHIN


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(24, 100), (150, 130)])
def test_many_small_steps_of_16_bit_parameters_are_kept(cuda_device, shape, dtype):
    """Steps and decay far below half a rounding step of the weights, against float64."""
    gen = torch.Generator(device=cuda_device).manual_seed(15)
    lr, decay, steps = 1e-4, 0.1, 120
    p = torch.nn.Parameter((0.02 * torch.randn(*shape, generator=gen, device=cuda_device)).to(dtype))
    w, m = p.detach().double(), torch.zeros(shape, dtype=torch.float64, device=cuda_device)
    start = w.clone()
    base = torch.randn(*shape, generator=gen, device=cuda_device)
    optimizer = Muon([p], lr=lr, weight_decay=decay)
    rate = lr * 0.2 * max(shape) ** 0.5
    moved = 0.0
    for _ in range(steps):
        p.grad = (base + 0.3 * torch.randn(*shape, generator=gen, device=cuda_device)).to(dtype)
        m.mul_(0.95).add_(p.grad.double())
        direction = _exact(p.grad.double() + 0.95 * m)
        w.mul_(1 - lr * decay).sub_(rate * direction)
        moved += rate * float(direction.norm())
        optimizer.step()
    # the weights' own rounding (half a step of the type), each direction's, and float32 sums
    room = 2.0 ** (-9 if dtype == torch.bfloat16 else -12) * float(w.norm()) * 1.01 + WITHIN * moved + steps * 2.0 ** -23 * float(w.norm())
    assert float((p.detach().double() - w).norm()) < room < 0.2 * float((w - start).norm())


def test_decay_alone_reaches_16_bit_parameters(cuda_device):
    p = torch.nn.Parameter(torch.full((16, 32), 0.02, dtype=torch.bfloat16, device=cuda_device))
    start = float(p.detach()[0, 0])
    optimizer = Muon([p], lr=1e-3, weight_decay=0.1)
    p.grad = torch.zeros_like(p)
    for _ in range(200):
        optimizer.step()
    want = start * (1 - 1e-4) ** 200
    assert bool(((p.detach().double() - want).abs() <= 2.0 ** -9 * want * 1.001).all())


def test_state_of_16_bit_parameters_survives_a_checkpoint(cuda_device):
    gen = torch.Generator(device=cuda_device).manual_seed(16)
    params = [torch.nn.Parameter(torch.randn(20, 40, generator=gen, device=cuda_device).bfloat16()) for _ in range(2)]
    optimizer = Muon(params, lr=1e-4)

    def step(optimizer, params, seed):
        gen = torch.Generator(device=cuda_device).manual_seed(seed)
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen, device=cuda_device).to(p.dtype)
        optimizer.step()

    for seed in range(3):
        step(optimizer, params, seed)
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    resumed = Muon(copies, lr=1e-4)
    resumed.load_state_dict(optimizer.state_dict())
    for seed in range(3, 12):
        step(optimizer, params, seed)
        step(resumed, copies, seed)
    for p, q in zip(params, copies):
        assert torch.equal(p, q)
        for name, value in optimizer.state[p].items():
            assert value.dtype == torch.float32 and torch.equal(value, resumed.state[q][name])


def test_a_16_bit_weight_changed_from_outside_keeps_its_new_value(cuda_device):
    p = torch.nn.Parameter(torch.full((16, 32), 0.02, dtype=torch.bfloat16, device=cuda_device))
    optimizer = Muon([p], lr=1e-3, weight_decay=0.1)
    p.grad = torch.zeros_like(p)
    optimizer.step()  # leaves a remainder of 2e-6
    changed = torch.linspace(0.0, 1e-4, 16 * 32, device=cuda_device).view(16, 32).bfloat16()
    p.data.copy_(changed)
    optimizer.param_groups[0]["lr"] = 0.0
    optimizer.step()
    assert torch.equal(p.detach(), changed)


def test_a_step_in_parts_is_the_step_at_once(cuda_device, monkeypatch):
    from moss_image_b200 import muon

    def run(limit):
        if limit is not None:
            monkeypatch.setattr(muon, "STEP_BYTES", limit)
        gen = torch.Generator(device=cuda_device).manual_seed(17)
        params = [torch.nn.Parameter(torch.randn(*s, generator=gen, device=cuda_device))
                  for s in [(200, 130)] * 5 + [(20, 300)] * 3 + [(1, 1)]]
        optimizer = Muon(params, lr=0.02, weight_decay=0.1)
        for _ in range(2):
            for p in params:
                p.grad = torch.randn(p.shape, generator=gen, device=cuda_device)
            optimizer.step()
        return params

    at_once, one_by_one = run(None), run(1)
    for a, b in zip(at_once, one_by_one):
        # the order of a matrix's sums may follow the size of its batch: one rounding of a direction to bfloat16
        assert float((a - b).detach().norm()) <= 2 * 0.004 * (a.shape[0] * a.shape[1]) ** 0.5 * 2.0 ** -8


def test_a_step_holds_a_bounded_share_of_memory(cuda_device):
    params = [torch.nn.Parameter(torch.zeros(2048, 2048, dtype=torch.bfloat16, device=cuda_device)) for _ in range(60)]
    for p in params:
        p.grad = torch.ones_like(p)
    optimizer = Muon(params)
    optimizer.step()  # the state exists after it
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(cuda_device)
    torch.cuda.reset_peak_memory_stats(cuda_device)
    optimizer.step()
    assert torch.cuda.max_memory_allocated(cuda_device) - before < 2 << 30


def test_a_refused_step_leaves_the_momentum(cuda_device):
    p = torch.nn.Parameter(torch.ones(8, 8, device=cuda_device))
    optimizer = Muon([p])
    p.grad = torch.ones_like(p)
    optimizer.step()
    held = {name: value.clone() for name, value in optimizer.state[p].items()}
    weight = p.detach().clone()
    for bad in (dict(steps=0), dict(eps=0.0), dict(coefficients=(40.0, 0.0, 0.0))):
        good = {name: optimizer.param_groups[0][name] for name in bad}
        optimizer.param_groups[0].update(bad)
        with pytest.raises(ValueError):
            optimizer.step()
        optimizer.param_groups[0].update(good)
        assert torch.equal(p.detach(), weight)
        assert all(torch.equal(value, optimizer.state[p][name]) for name, value in held.items())


def test_forward_mode_is_refused(cuda_device):
    from torch.autograd import forward_ad

    update = torch.randn(8, 12, device=cuda_device)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            orthogonalize(forward_ad.make_dual(update, torch.ones_like(update)))
        assert torch.equal(orthogonalize(update), orthogonalize(update))


def test_a_gradient_is_refused_and_the_values_stay(cuda_device):
    update = torch.randn(8, 12, device=cuda_device)
    tracked = update.clone().requires_grad_()
    direction = orthogonalize(tracked)
    assert torch.equal(direction.detach(), orthogonalize(update))
    with pytest.raises(NotImplementedError):
        (direction.float().sum() + tracked.sum()).backward()
    with torch.no_grad():
        assert not orthogonalize(tracked).requires_grad
    with pytest.raises(RuntimeError):
        orthogonalize(tracked, out=torch.empty(8, 12, dtype=torch.bfloat16, device=cuda_device))
