"""Checks of the paged cache's host side that need no GPU."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from cuda_b200 import paged


def test_tangents_are_refused():
    x, plain = torch.ones(3), torch.zeros(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        paged.no_grad_needed(plain)
        with pytest.raises(ValueError, match="tangent"):
            paged.no_grad_needed(plain, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
            paged.no_grad_needed(dual)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda v: paged.no_grad_needed(v) or v, (x,), (torch.ones(3),))
    paged.no_grad_needed(x)
