"""What the orthogonalising optimiser refuses before it touches a parameter or its state."""

from __future__ import annotations

import pytest
import torch

from moss_image_b200.muon import Muon

BAD = [dict(steps=0), dict(steps=17), dict(eps=0.0), dict(eps=float("inf")), dict(coefficients=(1.0, 2.0)),
       dict(coefficients=((1.0, 0.0, 0.0),) * 2), dict(coefficients=(40.0, 0.0, 0.0)),
       dict(coefficients=(float("nan"), 0.0, 0.0)), dict(lr=-1.0), dict(weight_decay=-0.1), dict(momentum=1.0)]


@pytest.mark.parametrize("bad", BAD)
def test_bad_options_are_refused_at_construction(bad):
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(4, 4))], **bad)


@pytest.mark.parametrize("bad", BAD)
def test_bad_options_of_a_group_are_refused_and_leave_no_group(bad):
    optimizer = Muon([torch.nn.Parameter(torch.zeros(4, 4))])
    with pytest.raises(ValueError):
        optimizer.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4, 4))], **bad))
    assert len(optimizer.param_groups) == 1


def test_unsupported_parameters_are_refused_at_construction():
    for wrong in (torch.zeros(4, 4, dtype=torch.float64), torch.zeros(4), torch.zeros(2, 4, 4)):
        with pytest.raises(ValueError):
            Muon([torch.nn.Parameter(wrong)])


def test_a_step_that_cannot_run_changes_nothing():
    p = torch.nn.Parameter(torch.ones(4, 4))
    optimizer = Muon([p])
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="CUDA"):
        optimizer.step()
    assert not optimizer.state[p] and torch.equal(p.detach(), torch.ones(4, 4))
    optimizer.param_groups[0]["steps"] = 0
    with pytest.raises(ValueError):
        optimizer.step()
    assert not optimizer.state[p]
