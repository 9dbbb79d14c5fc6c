"""Layer norm, coded activations and attention to another sequence where offsets pass 2^31 values: the far end of a tensor against
the same call on a copy of that end."""

from __future__ import annotations

import pytest
import torch

from moss_image_b200.activation_codes import coded_weight_gradient, decode_activation, encode_activation
from moss_image_b200.cross_attention import cross_attention
from moss_image_b200.norms import layer_norm
from moss_image_b200.quant_kernels import check_device_status

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
LAST = 100  # rows that are looked at


def _rows(dim, seed):
    """More than 2^31 values whose last rows are random."""
    x = torch.zeros(2 ** 31 // dim + 300, dim, device="cuda", dtype=BF16)
    x[-LAST:] = torch.randn(LAST, dim, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(BF16)
    return x


@pytest.mark.parametrize("dim", [16384, 4098])
def test_layer_norm(cuda_device, dim):
    x, grad = _rows(dim, 1), _rows(dim, 2)
    weight, bias = (torch.randn(dim, device="cuda").to(BF16) for _ in range(2))
    results = []
    for values, dy in ((x, grad), (x[-LAST:].clone(), grad[-LAST:].clone())):
        leaves = [t.detach().requires_grad_() for t in (values, weight, bias)]
        y = layer_norm(*leaves)
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        results.append((y.detach()[-LAST:].clone(), dx[-LAST:].clone(), dw, db))
        del y, dx, leaves
    assert all(torch.equal(a, b) for a, b in zip(results[0][:2], results[1][:2]))
    exact = torch.nn.functional.layer_norm(x[-LAST:].double(), (dim,), eps=1e-6)
    d = grad[-LAST:].double()
    # rows of zeros add nothing; f32 sums of 100 terms, one rounding
    for got, want, terms in ((results[0][2], (d * exact).sum(0), (d * exact).abs().sum(0)), (results[0][3], d.sum(0), d.abs().sum(0))):
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * terms).all()


@pytest.mark.parametrize("dim", [16384, 4098])
def test_codes(cuda_device, dim):
    x = _rows(dim, 3)
    coded = encode_activation(x)
    end = encode_activation(x[-LAST:].clone())
    assert torch.equal(coded.codes[-LAST:], end.codes) and torch.equal(coded.exponents[-LAST:], end.exponents)
    assert torch.equal(decode_activation(coded)[-LAST:], decode_activation(end))
    for features in (8, 40):
        dy = torch.randn(x.shape[0], features, device="cuda").to(BF16)
        got = coded_weight_gradient(dy, coded.codes, coded.exponents, torch.float32).double()
        near, d = decode_activation(end).double(), dy[-LAST:].double()
        assert ((got - d.t() @ near).abs() <= 2.0 ** -17 * (d.abs().t() @ near.abs())).all()
    check_device_status(x.device)


def test_attention(cuda_device):
    heads, dim = 128, 128
    many = 2 ** 31 // (heads * dim) + 200
    gen = torch.Generator(device="cuda").manual_seed(4)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(BF16)

    def step(q, k, v, grad, mask=None):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = cross_attention(*leaves, key_mask=mask)
        return [o.detach(), *torch.autograd.grad(o, leaves, grad)]

    # many queries, few keys
    q, k, v, grad = (torch.zeros(1, n, heads, dim, device="cuda", dtype=BF16) for n in (many, 5, 5, many))
    q[:, -LAST:], grad[:, -LAST:] = randn(1, LAST, heads, dim), randn(1, LAST, heads, dim)
    k.copy_(randn(*k.shape))
    v.copy_(randn(*v.shape))
    got = step(q, k, v, grad)
    end = step(q[:, -LAST:].clone(), k, v, grad[:, -LAST:].clone())
    assert all(torch.equal(a[:, -LAST:], b) for a, b in zip(got[:2], end[:2]))
    for a, b in zip(got[2:], end[2:]):  # rows whose gradient is zero add nothing; other splits, each result rounded once
        assert (a.double() - b.double()).norm() <= 2.0 ** -8 * b.double().norm()
    del got, q, grad
    # few queries, many keys, of which the last may be looked at
    q, grad = randn(1, 3, heads, dim), randn(1, 3, heads, dim)
    k, v = (torch.zeros(1, many, heads, dim, device="cuda", dtype=BF16) for _ in range(2))
    k[:, -LAST:], v[:, -LAST:] = randn(1, LAST, heads, dim), randn(1, LAST, heads, dim)
    mask = torch.arange(many, device="cuda")[None] >= many - LAST
    got = step(q, k, v, grad, mask)
    end = step(q, k[:, -LAST:].clone(), v[:, -LAST:].clone(), grad)
    assert not got[2][:, :-LAST].any() and not got[3][:, :-LAST].any()
    for a, b in zip((got[0], got[1], got[2][:, -LAST:], got[3][:, -LAST:]), end):  # keys fall into other tiles
        assert (a.double() - b.double()).norm() <= 2.0 ** -7 * b.double().norm()
    check_device_status(q.device)
