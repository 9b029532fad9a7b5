"""What the docstrings of a student's operators promise at the ends of their ranges, on the kernels."""
from __future__ import annotations

import pytest
import torch

import orda_ce_kernel as orda

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("width", [1 << 22, (1 << 22) + 1, 5_000_000])
def test_dropout_of_long_rows_that_are_not_dense(width):
    """Rows of 2^22 elements and more, as x, as the residual and as the gradient from above: the dense tensor's results."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(3, width, generator=g, device="cuda").to(BF)
    apart = torch.zeros(3, width + 5, dtype=BF, device="cuda")[:, 3:width + 3].copy_(x)
    across = x.t().contiguous().t()
    plain, both = orda.counter_dropout(x, 0.3, seed=9), orda.counter_dropout(x, 0.3, x, seed=9)
    for same in (apart, across):
        assert torch.equal(orda.counter_dropout(same, 0.3, seed=9), plain)
        assert torch.equal(orda.counter_dropout(x, 0.3, same, seed=9), both)
        leaf = x.detach().requires_grad_(True)
        (dx,) = torch.autograd.grad(orda.counter_dropout(leaf, 0.3, seed=9), leaf, same)
        assert torch.equal(dx, plain)
    row = x[:1].expand(3, width)
    assert torch.equal(orda.counter_dropout(row, 0.3, seed=9), orda.counter_dropout(row.contiguous(), 0.3, seed=9))
