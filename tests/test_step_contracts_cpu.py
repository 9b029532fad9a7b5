"""What the docstrings of a student's operators promise beside their formulas, on the CPU."""
from __future__ import annotations

import pytest
import torch

import orda_ce_kernel as orda


@pytest.mark.parametrize("call", [lambda x: orda.counter_dropout(x, 0.5), lambda x: orda.layer_norm(x, x[0], None, x, p=0.5)[1]],
                         ids=["dropout", "norm"])
def test_a_drawn_seed_does_not_depend_on_the_default_device(call):
    """seed=None draws from torch's CPU generator, inside torch.device() and out of it."""
    x = torch.randn(64, 64)
    torch.manual_seed(11)
    want, state = call(x), torch.get_rng_state()
    with torch.device("meta"):
        torch.manual_seed(11)
        assert torch.equal(call(x), want)
    assert torch.equal(torch.get_rng_state(), state)
