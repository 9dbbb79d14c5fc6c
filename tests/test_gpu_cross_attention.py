"""Attention to another sequence on the GPU against the formulas in float64.

Bounds, with h half a step of the 16-bit type and u = 2^-24. Forward: P is rounded to the type (h of each term), its
exponent is off by a few u times the logit's size and the hardware's exp2 by 2^-22, the sums by at most 2^-22 a step of 16 terms;
then one rounding. So |O - exact| <= (1.1 h + e) sum_j P_j |V_j| + h |O|, where e is the relative error of an exponential.
Backward: dS is rounded once (h), P in dV once; delta is taken from the rounded O and adds h sum|O dO| to every dS / P.
float16 rounds values below 2^-14 to multiples of 2^-24, so that dS may be off by another f = 2^-25 each; the exponentials are
lifted by 2^7 in the forward pass (a row's sum is then at least 2^7) and P by 2^14 in dV, which leaves f 2^-14 of each there.
"""

from __future__ import annotations

import math

import pytest
import torch

from moss_image_b200.cross_attention import cross_attention, cross_attention_packed
from moss_image_b200.packed import cumulative_lengths
from moss_image_b200.quant_kernels import check_device_status

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
HALF_STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def _least(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _exact(q, k, v, allowed, scale, grad=None):
    """(result, bound) pairs of O and, with a gradient, dQ, dK, dV, from float64; [batch, tokens, heads, dim] in and out."""
    dtype = q.dtype
    h, groups = HALF_STEP[dtype], q.shape[2] // k.shape[2]
    q, k, v = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    k_all, v_all = (t.repeat_interleave(groups, 1) for t in (k, v))
    logits = scale * (q @ k_all.mT)
    if allowed is not None:
        logits = logits.masked_fill(~allowed, -math.inf)
    top = logits.amax(-1, keepdim=True).clamp_min(-1e300)
    p = torch.exp(logits - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    # the logits' own f32 sums, their distance from the row's reference, exp2 itself, and the sums over keys
    reach = scale * (q.abs() @ k_all.abs().mT).amax(-1, keepdim=True)
    e = 2.0 ** -21 * (4 + reach) + (k.shape[2] / 16 + 8) * 2.0 ** -22
    o = p @ v_all
    spread = p @ v_all.abs()
    floor = 2.0 ** -25 if dtype == F16 else 0.0
    seen = torch.ones_like(logits) if allowed is None else allowed.expand_as(logits).double()
    o_off = (1.1 * h + e) * spread + 2.0 ** -7 * floor * (seen @ v_all.abs())
    results = [(o, o_off)]
    if grad is not None:
        g = grad.detach().double().transpose(1, 2)
        dp = g @ v_all.mT
        delta = (g * o).sum(-1, keepdim=True)
        rows = (g.abs() * ((h + 1.1 * h + e) * spread + h * o.abs())).sum(-1, keepdim=True)  # of delta, through the rounded O
        dp_size = g.abs() @ v_all.abs().mT
        ds = p * (dp - delta)
        ds_off = (1.1 * h + e) * ds.abs() + p * (rows + (8 + q.shape[-1] / 16) * 2.0 ** -22 * (dp_size + spread.mul(g.abs()).sum(-1, keepdim=True)))
        ds_off = ds_off + floor * seen
        tail = (max(q.shape[2], k.shape[2]) * groups / 16 + 16) * 2.0 ** -22

        def fold(t):
            return t.unflatten(1, (-1, groups)).sum(2)

        results.append((scale * (ds @ k_all), scale * (ds_off @ k_all.abs() + tail * (ds.abs() @ k_all.abs()))))
        results.append((fold(scale * (ds.mT @ q)), fold(scale * (ds_off.mT @ q.abs() + tail * (ds.abs().mT @ q.abs())))))
        results.append((fold(p.mT @ g), fold(((1.1 * h + e + tail) * p + 2.0 ** -14 * floor * seen).mT @ g.abs())))
    return [(r.transpose(1, 2), b.transpose(1, 2)) for r, b in results]


def _assert_near(names, got, expected):
    for name, value, (exact, slack) in zip(names, got, expected):
        allowed = slack + HALF_STEP[value.dtype] * (exact.abs() + slack) + _least(value.dtype)
        worst = ((value.double() - exact).abs() / allowed).max().item() if value.numel() else 0.0
        assert worst <= 1.0, f"{name}: {worst:.3f} of what rounding allows"


def _tensors(batch, tq, tk, hq, hk, dim, dtype, seed=0, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return (size * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)

    return randn(batch, tq, hq, dim), randn(batch, tk, hk, dim), randn(batch, tk, hk, dim), randn(batch, tq, hq, dim)


def _run(q, k, v, grad, **options):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*leaves, **options)
    got = [o.detach(), *torch.autograd.grad(o, leaves, grad)]
    check_device_status(q.device)
    with torch.no_grad():
        assert torch.equal(cross_attention(q, k, v, **options), got[0])
    return got


def _check(q, k, v, grad, mask=None, scale=None):
    got = _run(q, k, v, grad, key_mask=mask, scale=scale)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    allowed = None if mask is None else mask[:, None, None]
    _assert_near(("o", "dq", "dk", "dv"), got, _exact(q, k, v, allowed, scale, grad))
    return got


SHAPES = [  # batch, query tokens, key tokens, query heads, key heads, head_dim
    (1, 1, 1, 1, 1, 8), (2, 1, 2, 2, 1, 64), (1, 3, 127, 2, 2, 16), (1, 128, 128, 1, 1, 64), (2, 129, 128, 2, 2, 128),
    (1, 255, 129, 3, 1, 72), (1, 256, 257, 2, 2, 40), (3, 300, 77, 4, 2, 80), (1, 513, 640, 2, 1, 128), (2, 1000, 300, 6, 2, 64),
    (1, 2, 2050, 2, 1, 96), (1, 1, 4096, 1, 1, 128), (1, 4500, 5, 1, 1, 120), (4, 1, 512, 24, 24, 128), (1, 5000, 260, 8, 1, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_formulas(cuda_device, shape, dtype):
    _check(*_tensors(*shape, dtype, sum(shape)))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_logits_move_the_reference(cuda_device, dtype):
    q, k, v, grad = _tensors(1, 200, 900, 2, 2, 64, dtype, 1)
    k[:, 400:] *= 6.0  # later keys lift the rows' maximum by more than 2^8
    k[:, 800:] *= 2.0
    _check(q, k, v, grad, scale=0.3)
    _check(q, k.flip(1), v, grad, scale=0.3)
    _check(q, k, v, grad, scale=1e-6)


def _masks(batch, tk):
    lengths = torch.tensor([(0, tk, 1, tk // 2, tk - 1, 129)[i % 6] for i in range(batch)], device="cuda")
    prefix = torch.arange(tk, device="cuda")[None] < lengths[:, None]
    gen = torch.Generator(device="cuda").manual_seed(5)
    holes = torch.rand(batch, tk, generator=gen, device="cuda") < 0.5
    late = torch.zeros(batch, tk, dtype=torch.bool, device="cuda")
    late[:, -1] = True
    late[0] = False
    middle = torch.zeros_like(late)
    middle[:, tk // 3 : tk // 3 + 140] = True  # whole tiles without keys on both sides
    return {"prefix": prefix, "holes": holes, "late": late, "middle": middle}


@pytest.mark.parametrize("kind", ["prefix", "holes", "late", "middle"])
@pytest.mark.parametrize("batch,tq,tk,hq,hk,dim,dtype", [(6, 130, 300, 2, 1, 64, BF16), (6, 70, 513, 2, 2, 128, F16),
                                                         (6, 2, 1100, 1, 1, 80, BF16)])
def test_masks(cuda_device, kind, batch, tq, tk, hq, hk, dim, dtype):
    mask = _masks(batch, tk)[kind]
    got = _check(*_tensors(batch, tq, tk, hq, hk, dim, dtype, 2), mask=mask)
    nothing = ~mask.any(1)
    assert not any(t[nothing].any() for t in got)
    assert not got[2][~mask].any() and not got[3][~mask].any()


def test_masks_of_many_tiles(cuda_device):
    mask = torch.rand(9, 4000, device="cuda") < 0.02  # 9 x 32 tiles
    mask[:, 1000:2500] = False
    _check(*_tensors(9, 33, 4000, 1, 1, 64, BF16, 3), mask=mask)


@pytest.mark.parametrize("dim", [64, 128])
def test_what_lies_in_masked_places_is_not_read(cuda_device, dim):
    q, k, v, grad = _tensors(4, 150, 400, 2, 2, dim, BF16, 4)
    mask = _masks(4, 400)["holes"]
    mask[2] = False
    clean = _run(q, k, v, grad, key_mask=mask)
    for poison in (float("nan"), float("inf"), -float("inf")):
        k2, v2 = k.clone(), v.clone()
        k2[~mask] = poison
        v2[~mask] = poison
        assert all(torch.equal(a, b) for a, b in zip(_run(q, k2, v2, grad, key_mask=mask), clean))


def test_non_finite_values_where_they_are_looked_at(cuda_device):
    q, k, v, _ = _tensors(2, 40, 200, 2, 2, 64, BF16, 5)
    clean = cross_attention(q, k, v)
    v[1, 7, 0, 3] = float("nan")
    q[0, 5, 1, 2] = float("nan")
    o = cross_attention(q, k, v)
    assert o[1, :, 0, 3].isnan().all() and o[0, 5, 1].isnan().all()
    o[1, :, 0, 3], o[0, 5, 1] = clean[1, :, 0, 3], clean[0, 5, 1]
    assert torch.equal(o, clean)


def test_one_key_leaves_no_gradient_of_its_logit(cuda_device):
    q, k, v, grad = _tensors(2, 50, 300, 2, 1, 64, BF16, 6)
    mask = torch.zeros(2, 300, dtype=torch.bool, device="cuda")
    mask[:, 260] = True
    for args, options in (((q, k[:, :1], v[:, :1], grad), {}), ((q, k, v, grad), {"key_mask": mask})):
        got = _run(*args, **options)
        assert not got[1].any() and not got[2].any()


def test_views_strides_and_copies(cuda_device):
    q, k, v, grad = _tensors(2, 140, 90, 4, 2, 72, BF16, 7)
    plain = _check(q, k, v, grad)
    fused = torch.stack((k, v), 2)  # keys and values of one projection
    by_heads = q.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(2, 90, 2, 73, dtype=BF16, device="cuda")[..., :72].copy_(k)  # rows off the 16-byte grid
    shifted = torch.empty(1 + v.numel(), dtype=BF16, device="cuda")[1:].view_as(v).copy_(v)
    for views in ((q, fused[:, :, 0], fused[:, :, 1]), (by_heads, k, v), (q, odd, shifted)):
        assert all(torch.equal(a, b) for a, b in zip(_run(*views, grad), plain))
    strided = torch.empty(2, 140, 4, 144, dtype=BF16, device="cuda")[..., ::2].copy_(grad)
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, strided), plain))
    off = torch.empty(1 + grad.numel(), dtype=BF16, device="cuda")[1:].view_as(grad).copy_(grad)
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, off), plain))
    # one caption for the whole batch: an expanded dimension, whose gradient is summed by autograd
    one_k, one_v = k[:1].detach().requires_grad_(), v[:1].detach().requires_grad_()
    o = cross_attention(q, one_k.expand(2, -1, -1, -1), one_v.expand(2, -1, -1, -1))
    dk, = torch.autograd.grad(o, one_k, grad)
    parts = _run(q, k[:1].repeat(2, 1, 1, 1), v[:1].repeat(2, 1, 1, 1), grad)
    assert torch.equal(o, parts[0]) and torch.equal(dk, parts[2].sum(0, keepdim=True))
    mask = torch.zeros(2, 180, dtype=torch.bool, device="cuda")[:, ::2]
    mask[:, :50] = True
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, grad, key_mask=mask), _run(q, k, v, grad, key_mask=mask.contiguous())))
    row = torch.ones(1, 90, dtype=torch.bool, device="cuda").expand(2, -1)
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, grad, key_mask=row), plain))


def test_only_the_gradients_that_are_asked_for(cuda_device):
    tensors = _tensors(2, 140, 300, 4, 2, 64, BF16, 8)
    q, k, v, grad = tensors
    full = _run(q, k, v, grad)
    for wanted in ((0,), (1,), (2,), (0, 2)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        for i, part in zip(wanted, torch.autograd.grad(cross_attention(*leaves), [leaves[i] for i in wanted], grad)):
            assert torch.equal(part, full[1 + i])


def test_gradient_against_differences(cuda_device):
    q, k, v, grad = _tensors(1, 9, 20, 2, 1, 16, F16, 9)
    got = _run(q, k, v, grad)

    def loss(values):
        a, b, c = (t.transpose(1, 2) for t in values)
        p = torch.softmax(0.25 * a @ b.repeat_interleave(2, 1).mT, -1)
        return ((p @ c.repeat_interleave(2, 1)).transpose(1, 2) * grad.double()).sum()

    points = [t.double() for t in (q, k, v)]
    for i, part in enumerate(got[1:]):
        step = torch.randn_like(points[i])
        moved = [[t + s * 1e-5 * step if n == i else t for n, t in enumerate(points)] for s in (1, -1)]
        slope = (loss(moved[0]) - loss(moved[1])) / 2e-5
        bound = _exact(q, k, v, None, 0.25, grad)[1 + i]
        allowed = ((bound[1] + HALF_STEP[F16] * (bound[0].abs() + bound[1])) * step.abs()).sum() + 1e-6 * slope.abs()
        assert abs((part.double() * step).sum() - slope) <= allowed


# ------------------------------------------------------------------------------------------ packed
def _packed(lengths_q, lengths_k, hq, hk, dim, dtype, seed=0, behind=0):
    q, k, v, grad = (t[0] for t in _tensors(1, sum(lengths_q) + behind, sum(lengths_k) + behind, hq, hk, dim, dtype, seed))
    return q, k, v, grad, cumulative_lengths(lengths_q, q.device), cumulative_lengths(lengths_k, q.device)


def _run_packed(q, k, v, grad, q_offsets, k_offsets):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention_packed(*leaves, q_offsets, k_offsets)
    got = [o.detach(), *torch.autograd.grad(o, leaves, grad)]
    check_device_status(q.device)
    return got


@pytest.mark.parametrize("lengths_q,lengths_k,hq,hk,dim,dtype", [
    ([5], [7], 1, 1, 64, BF16),
    ([1, 300, 128, 17], [130, 1, 77, 128], 2, 1, 64, F16),
    ([200, 0, 33, 1], [50, 20, 0, 300], 4, 2, 128, BF16),  # empty on either side
    ([0, 0, 9], [0, 5, 0], 2, 2, 80, BF16),
    ([3] * 70, [11] * 70, 1, 1, 64, F16),  # more sequences than a warp has lanes
    ([1000, 1, 500], [200, 600, 90], 3, 3, 128, F16),
    ([2, 1], [1500, 900], 2, 1, 64, BF16),  # keys split
])
def test_packed_sequences(cuda_device, lengths_q, lengths_k, hq, hk, dim, dtype):
    behind = 5
    q, k, v, grad, q_offsets, k_offsets = _packed(lengths_q, lengths_k, hq, hk, dim, dtype, 1, behind)
    got = _run_packed(q, k, v, grad, q_offsets, k_offsets)
    starts = [[sum(n[:i]) for i in range(len(n) + 1)] for n in (lengths_q, lengths_k)]
    for s, (nq, nk) in enumerate(zip(lengths_q, lengths_k)):
        rows, keys = slice(starts[0][s], starts[0][s] + nq), slice(starts[1][s], starts[1][s] + nk)
        parts = [got[0][rows], got[1][rows], got[2][keys], got[3][keys]]
        if nq == 0 or nk == 0:
            assert not any(p.any() for p in parts)
            continue
        _assert_near(("o", "dq", "dk", "dv"), [p[None] for p in parts],
                     _exact(q[None, rows], k[None, keys], v[None, keys], None, dim ** -0.5, grad[None, rows]))
    assert not any(t[-behind:].any() for t in got)  # rows behind the last sequence


def test_packed_neighbours_do_not_leak(cuda_device):
    q, k, v, grad, q_offsets, k_offsets = _packed([100, 60, 200], [70, 150, 40], 2, 2, 64, BF16, 2, 9)
    clean = _run_packed(q, k, v, grad, q_offsets, k_offsets)
    for t, start, end in ((q, 100, 160), (grad, 100, 160), (k, 70, 220), (v, 70, 220)):
        t[start:end] = float("nan")
        t[-9:] = float("inf")
    dirty = _run_packed(q, k, v, grad, q_offsets, k_offsets)
    for a, b, start, end in zip(dirty, clean, (100, 100, 70, 70), (160, 160, 220, 220)):
        assert torch.equal(a[:start], b[:start]) and torch.equal(a[end:], b[end:])


def test_packed_agrees_with_batches(cuda_device):
    q, k, v, grad = _tensors(3, 140, 130, 4, 2, 64, BF16, 3)
    plain = _run(q, k, v, grad)
    offsets = [cumulative_lengths([n] * 3, q.device) for n in (140, 130)]
    got = _run_packed(*(t.flatten(0, 1) for t in (q, k, v, grad)), *offsets)
    assert torch.equal(got[0], plain[0].flatten(0, 1))
    for a, b in zip(got[1:], plain[1:]):  # the splits may differ, and with them the order of sums
        assert (a - b.flatten(0, 1)).abs().max() <= 2 * HALF_STEP[BF16] * b.abs().max()


def test_boundaries_outside_the_rows_stay_in_bounds(cuda_device):
    q, k, v, grad, _, _ = _packed([40], [30], 1, 1, 64, BF16, 4)
    wild = torch.tensor([0, 10, 1 << 40], device="cuda")
    falling = torch.tensor([0, 25, -7], device="cuda")
    o = cross_attention_packed(q, k, v, wild, falling)
    torch.cuda.synchronize()
    assert o.shape == q.shape


# ------------------------------------------------------------------------------------------ life
def test_no_tokens(cuda_device):
    q, k, v, grad = _tensors(2, 10, 12, 2, 1, 64, BF16, 5)
    o, dq, dk, dv = _run(q, k[:, :0], v[:, :0], grad)
    assert not o.any() and not dq.any() and dk.shape == (2, 0, 1, 64)
    o, dq, dk, dv = _run(q[:, :0], k, v, grad[:, :0])
    assert o.shape == (2, 0, 2, 64) and not dk.any() and not dv.any()
    assert cross_attention(q[:0], k[:0], v[:0]).shape == (0, 10, 2, 64)


def test_same_bits_on_side_streams_and_in_graphs(cuda_device):
    q, k, v, grad = _tensors(2, 700, 400, 4, 2, 64, BF16, 6)
    mask = _masks(2, 400)["holes"]
    thin = q[:, :1].contiguous()

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = cross_attention(*leaves, key_mask=mask)
        return [o.detach(), *torch.autograd.grad(o, leaves, grad), cross_attention(thin, k, v)]

    first = step()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for stream in streams:  # two calls at once
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            outs.append(step())
    for stream in streams:
        torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for out in outs for a, b in zip(first, out))
    graphs, captured = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            captured.append(step())
    mask.copy_(_masks(2, 400)["prefix"])
    v.mul_(0.5)
    for graph in graphs:
        graph.replay()
    fresh = step()
    assert all(torch.equal(a, b) for out in captured for a, b in zip(fresh, out))
    check_device_status(q.device)


def test_refusals(cuda_device):
    q, k, v, _ = _tensors(2, 10, 12, 4, 2, 64, BF16, 7)
    offsets = torch.tensor([0, 5, 10], device="cuda")
    bad = [
        (lambda: cross_attention(q, k, v.float()), "one dtype"),
        (lambda: cross_attention(q.float(), k.float(), v.float()), "float16 or bfloat16"),
        (lambda: cross_attention(q, k.cpu(), v), "one device"),
        (lambda: cross_attention(q, k[:, :11], v), "one shape"),
        (lambda: cross_attention(q, k[:1], v[:1]), "batch"),
        (lambda: cross_attention(q[..., :60], k[..., :60], v[..., :60]), "multiple of 8"),
        (lambda: cross_attention(*(torch.cat([t] * 3, -1) for t in (q, k, v))), "up to 128"),
        (lambda: cross_attention(q[:, :, :3], k, v), "multiple of the key"),
        (lambda: cross_attention(q[0], k[0], v[0]), "batch, tokens"),
        (lambda: cross_attention(q, k, v, scale=-1.0), "positive"),
        (lambda: cross_attention(q, k, v, scale=math.inf), "finite"),
        (lambda: cross_attention(q, k, v, key_mask=torch.ones(2, 12, device="cuda")), "bool"),
        (lambda: cross_attention(q, k, v, key_mask=torch.ones(2, 11, dtype=torch.bool, device="cuda")), "k_tokens"),
        (lambda: cross_attention_packed(q[0], k[0], v[0], offsets.int(), offsets), "int64"),
        (lambda: cross_attention_packed(q[0], k[0], v[0], offsets, offsets[:2]), "same sequences"),
        (lambda: cross_attention_packed(q[0], k[0], v[0], offsets.cpu(), offsets), "device"),
        (lambda: cross_attention_packed(q, k, v, offsets, offsets), "tokens, heads"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    leaf = q.detach().requires_grad_()
    slope, = torch.autograd.grad(cross_attention(leaf, k, v).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(slope.float().sum(), leaf)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            cross_attention(torch.autograd.forward_ad.make_dual(q, q), k, v)


# ------------------------------------------------------------------------------------------ NaN and infinities that are looked at
def _run_with_nan(q, k, v, grad, **options):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*leaves, **options)
    got = [o.detach(), *torch.autograd.grad(o, leaves, grad)]
    check_device_status(q.device)
    return got


def _assert_non_finite_as_defined(q, k, v, grad, mask, poisoned, head):
    """NaN where the formulas have it, in float64, and nowhere else; other heads as without the poison; what stays finite of the
    poisoned one is within its bounds (there the poisoned key's weight is zero)."""
    scale = q.shape[-1] ** -0.5
    allowed = torch.ones(q.shape[0], k.shape[1], dtype=torch.bool, device="cuda") if mask is None else mask
    got = _run_with_nan(q, k, v, grad, key_mask=mask)
    with_poison = _exact(q, k, v, allowed[:, None, None], scale, grad)
    calm, left = k.clone(), allowed.clone()
    calm[:, poisoned, head] = 0.0
    left[:, poisoned] = False
    without = _exact(q, calm, v, left[:, None, None], scale, grad)
    clean = _run(q, calm, v, grad, key_mask=mask)
    for part in (*with_poison[2:], *without[2:]):
        part[0][~allowed] = 0.0  # a key that may not be looked at has no gradient, whatever the others hold
    for name, value, (exact, _), (near, slack), other in zip(("o", "dq", "dk", "dv"), got, with_poison, without, clean):
        assert torch.equal(value.isnan(), exact.isnan()), name
        good = ~exact.isnan()
        good[:, :, [h for h in range(value.shape[2]) if h != head]] = False
        bound = slack + HALF_STEP[value.dtype] * (near.abs() + slack) + _least(value.dtype)
        assert ((value.double() - near).abs()[good] <= bound[good]).all(), name
        rest = [h for h in range(value.shape[2]) if h != head]
        assert torch.equal(value[:, :, rest], other[:, :, rest]), name


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
def test_non_finite_keys_that_are_looked_at(cuda_device, dim, dtype, masked):
    q, k, v, grad = _tensors(1, 130, 140, 2, 2, dim, dtype, 11)
    mask = None
    if masked:  # a key that may not be looked at in the poisoned half tile
        mask = torch.ones(1, 140, dtype=torch.bool, device="cuda")
        mask[:, 20] = False
    for key in (*range(12), 63, 139):
        for poison in (float("nan"), float("inf"), -float("inf")):
            bad = k.clone()
            bad[0, key, 0, 5] = poison  # logits of both signs where it is an infinity
            _assert_non_finite_as_defined(q, bad, v, grad, mask, [key], 0)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tq,tk", [(130, 140), (1, 1024)])  # whole, and with the keys split
def test_two_nan_keys_are_not_a_row_without_keys(cuda_device, tq, tk, dtype):
    q, k, v, grad = _tensors(1, tq, tk, 1, 1, 64, dtype, 12)
    k[0, 4], k[0, 5] = float("nan"), float("nan")
    assert all(t.isnan().all() for t in _run_with_nan(q, k, v, grad))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("tq,tk", [(130, 140), (1, 1024)])
def test_logits_of_minus_infinity_weigh_nothing(cuda_device, tq, tk, dtype):
    q, k, v, grad = _tensors(1, tq, tk, 1, 1, 64, dtype, 13)
    q[..., 3] = q[..., 3].abs() + 0.125
    k[..., 3] = -float("inf")
    o, dq, dk, dv = _run_with_nan(q, k, v, grad)
    assert not o.any() and not dk.any() and not dv.any()
    assert dq[..., 3].isnan().all() and not dq[..., :3].any() and not dq[..., 4:].any()  # 0 * inf


@pytest.mark.parametrize("masked", [False, True])
def test_one_key_keeps_nan_in_its_gradients(cuda_device, masked):
    tensors = _tensors(1, 50, 300 if masked else 1, 1, 1, 64, BF16, 14)
    at = 260 if masked else 0
    mask = None
    if masked:
        mask = torch.zeros(1, 300, dtype=torch.bool, device="cuda")
        mask[:, at] = True
    for which, place in ((0, (0, 5)), (1, (0, at)), (2, (0, at, 0, 3)), (3, (0, 5))):  # in q, k, v and the gradient of o
        bad = [t.clone() for t in tensors]
        bad[which][place] = float("nan")
        q, k, v, grad = bad
        dq, dk = (t.isnan() for t in _run_with_nan(q, k, v, grad, key_mask=mask)[1:3])
        rows = torch.zeros(1, 50, 1, 64, dtype=torch.bool, device="cuda")
        rows[(0, 5) if which in (0, 3) else ...] = True  # whose logit's gradient is NaN
        assert torch.equal(dq, rows)
        assert dk[0, at].all()
        if which != 0:  # (the sum dS^T Q has the NaN of Q whatever dS is)
            assert dk.sum() == 64


@pytest.mark.parametrize("batch,tk", [(65, 400), (1, 33000)])  # masks of more than 256 tiles
def test_one_key_in_masks_of_many_tiles(cuda_device, batch, tk):
    q, k, v, grad = _tensors(batch, 3, tk, 1, 1, 64, BF16, 15)
    mask = torch.zeros(batch, tk, dtype=torch.bool, device="cuda")
    at = torch.arange(batch, device="cuda") * 61 % tk if batch > 1 else torch.tensor([tk - 200], device="cuda")
    mask[torch.arange(batch, device="cuda"), at] = True
    o, dq, dk, dv = _run(q, k, v, grad, key_mask=mask)
    assert torch.equal(o, v[mask][:, None].expand_as(o)) and not dq.any() and not dk.any()
    mask[-1, (int(at[-1]) + 150) % tk] = True  # a second key for one of them
    _check(q, k, v, grad, mask=mask)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, F16)])
@pytest.mark.parametrize("tk", [5, 100, 130])
def test_many_units_of_few_keys(cuda_device, tk, dim, dtype):
    """A multiprocessor's units follow one another within a microsecond or two, thousands of them in a row."""
    q, k, v, grad = _tensors(1, 20000, tk, 48, 48, dim, dtype, 16)
    rows = torch.randint(0, 20000, (40,), device="cuda")
    mask = torch.rand(1, tk, device="cuda") < 0.5
    for options in ({}, {"key_mask": mask}):
        first = _run(q, k, v, grad, **options)
        for _ in range(12):
            with torch.no_grad():
                assert torch.equal(cross_attention(q, k, v, **options), first[0])
        check_device_status(q.device)
        allowed = None if not options else mask[:, None, None]
        _assert_near(("o", "dq"), [t[:, rows] for t in first[:2]],
                     _exact(q[:, rows], k, v, allowed, dim ** -0.5, grad[:, rows])[:2])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["dense", "masked", "packed"])
@pytest.mark.parametrize("keys", [2, 4, 9, 30, 128])
def test_gradients_of_short_captions_have_two_roundings(cuda_device, keys, layout, dtype):
    """A value's rounding is off by h / sqrt(3) / m in the mean, m in [1, 2) its mantissa: 0.425 h over values of all sizes. dQ and dK
    have that of dS and their own, 0.6 h, and a tenth of that for the sample; not that of O, which delta could be taken from."""
    batch, tq, heads, dim = 3, 500, 4, 64
    q, k, v, grad = _tensors(batch, tq, 140 if layout == "masked" else keys, heads, heads, dim, dtype, 18)
    allowed = None
    if layout == "packed":
        offsets = [cumulative_lengths([n] * batch, q.device) for n in (tq, keys)]
        got = [t.unflatten(0, (batch, -1)) for t in _run_packed(*(t.flatten(0, 1) for t in (q, k, v, grad)), *offsets)]
    elif layout == "masked":
        mask = torch.zeros(batch, 140, dtype=torch.bool, device="cuda")
        mask[:, : 2 * keys : 2] = True
        mask[:, 128:] = False
        allowed = mask[:, None, None]
        got = _run(q, k, v, grad, key_mask=mask)
    else:
        got = _run(q, k, v, grad)
    for name, value, (exact, _) in zip(("dq", "dk"), got[1:], _exact(q, k, v, allowed, dim ** -0.5, grad)[1:]):
        assert (value.double() - exact).norm() <= 0.66 * HALF_STEP[dtype] * exact.norm(), name
