"""Rotary angles on the CPU: frequencies, their scalings, the table, and the device refusal."""

from __future__ import annotations

import math

import pytest
import torch

from moss_image_b200.rotary import apply_rotary, rotary_frequencies, rotary_table, yarn_magnitude


def test_frequencies_are_powers_of_the_base():
    got = rotary_frequencies(8, theta=100.0)
    want = torch.tensor([100.0 ** (-i / 4) for i in range(4)], dtype=torch.float64)
    assert torch.allclose(got, want, rtol=1e-14, atol=0.0)


def test_linear_scaling_divides_every_frequency():
    assert torch.allclose(rotary_frequencies(16, scaling="linear", factor=4.0) * 4.0, rotary_frequencies(16), rtol=1e-14)


def test_ntk_scaling_keeps_the_fastest_and_divides_the_slowest():
    plain, scaled = rotary_frequencies(64), rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert scaled[0] == plain[0]
    assert math.isclose(float(plain[-1] / scaled[-1]), 8.0, rel_tol=1e-12)
    assert bool((scaled <= plain).all())


def test_yarn_scaling_keeps_fast_pairs_and_divides_slow_ones():
    plain = rotary_frequencies(128)
    scaled = rotary_frequencies(128, scaling="yarn", factor=8.0, original_length=4096)
    ratio = plain / scaled
    turns = 4096 * plain / (2 * math.pi)
    assert torch.allclose(ratio[turns > 40.0], torch.ones(()).double())
    assert torch.allclose(ratio[turns < 0.8], torch.full((), 8.0).double())
    assert bool((ratio[1:] >= ratio[:-1] - 1e-12).all())
    assert yarn_magnitude(1.0) == 1.0 and math.isclose(yarn_magnitude(math.e), 1.1)


def test_table_keeps_the_angle_of_a_far_position():
    place = 10_000_019
    cos, sin = rotary_table(torch.tensor([place]), rotary_frequencies(4))
    for pair, frequency in enumerate((1.0, 0.01)):
        assert abs(float(cos[0, pair]) - math.cos(place * frequency)) < 1e-6
        assert abs(float(sin[0, pair]) - math.sin(place * frequency)) < 1e-6


def test_table_of_axes_puts_their_pairs_one_after_another():
    places = torch.tensor([[0, 3, 5], [2, 1, 4]])
    vectors = [rotary_frequencies(4), rotary_frequencies(6), rotary_frequencies(2)]
    cos, sin = rotary_table(places, vectors, magnitude=1.5)
    assert cos.shape == (2, 6) and cos.dtype == torch.float32
    parts = [rotary_table(places[:, axis], vector) for axis, vector in enumerate(vectors)]
    assert torch.allclose(cos, 1.5 * torch.cat([c for c, _ in parts], 1))
    assert torch.allclose(sin, 1.5 * torch.cat([s for _, s in parts], 1))


@pytest.mark.parametrize("arguments", [
    dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, theta=0.0), dict(dim=8, factor=0.5),
    dict(dim=8, scaling="yarn", factor=2.0),
])
def test_frequencies_refuse(arguments):
    with pytest.raises(ValueError):
        rotary_frequencies(**arguments)


def test_table_refuses_positions_without_a_vector_for_each_axis():
    with pytest.raises(ValueError):
        rotary_table(torch.zeros(3, 2), rotary_frequencies(4))
    with pytest.raises(ValueError):
        rotary_table(torch.zeros(3, 2, 1), rotary_frequencies(4))


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 1, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        apply_rotary(q, q, torch.zeros(2, 2), torch.zeros(2, 2))


@pytest.mark.parametrize("theta,length", [(1e4, 131072), (256.0, 4096), (500.0, 32768), (1e4, 2048), (1e6, 40)])
def test_yarn_divides_wholly_only_pairs_that_turn_too_rarely(theta, length):
    """Pair by pair: the divisor follows the pair's index between the ends of the ramp, which lie where
    the turns pass the two betas, past the last pair too."""
    factor, half = 8.0, 64
    plain = rotary_frequencies(2 * half, theta=theta)
    ratio = plain / rotary_frequencies(2 * half, theta=theta, scaling="yarn", factor=factor, original_length=length)
    turns = length * plain / (2 * math.pi)
    assert bool((ratio[turns > 1.001] < factor * (1 - 1e-9)).all())
    low, high = (half * math.log(length / (beta * 2 * math.pi)) / math.log(theta) for beta in (32.0, 1.0))
    low = max(math.floor(low), 0)
    high = math.ceil(high)
    for pair in range(half):
        part = min(max((pair - low) / max(high - low, 1e-3), 0.0), 1.0)
        assert math.isclose(float(1.0 / ratio[pair]), (1.0 - part) + part / factor, rel_tol=1e-9)
