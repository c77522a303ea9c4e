"""Muon's host side on the CPU: what its constructor refuses."""

import math

import pytest
import torch

from training.optim import Muon


@pytest.mark.parametrize("match, kw", [
    ("steps", dict(steps=65)), ("coefficients", dict(coefficients=(1.5, -0.5))),
    ("coefficients", dict(coefficients=(3.0, math.nan, 2.0))),
    ("coefficients", dict(coefficients=(3.0, -4.0, math.inf))),
])
def test_what_the_iteration_refuses_is_refused_at_construction(match, kw):
    """In step() it would come after the momentum has moved."""
    with pytest.raises(ValueError, match=match):
        Muon([torch.zeros(4, 6, requires_grad=True)], **kw)


def test_bounds_of_the_iteration_are_taken():
    for kw in (dict(steps=1), dict(steps=64), dict(coefficients=[1.5, -0.5, 0.0])):
        opt = Muon([torch.zeros(4, 6, requires_grad=True)], **kw)
        assert opt.steps == kw.get("steps", 5) and len(opt.coefficients) == 3
