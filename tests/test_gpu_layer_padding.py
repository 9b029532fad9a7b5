"""Infinities beside the padding of the feed-forward block: h, da and db lie in rows whose length is the inner width rounded
up, and what stands behind the inner width reaches no result."""
from __future__ import annotations

import pytest
import torch

import orda_ce_kernel as orda
from tests.test_gpu_layers import DTYPES

pytestmark = pytest.mark.gpu


def positive(*shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.rand(shape, generator=g) * 0.25 + 0.0625).to(dtype).cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [4, 40, 300])
@pytest.mark.parametrize("inner", [100, 102, 129])
def test_an_infinite_row_of_x(inner, N, dtype):
    """All weights positive: an infinity in x makes a, b, h and y of its row infinite, by the formulas; without padding
    nothing is NaN."""
    x, wg, wu, wd = (positive(*s, dtype=dtype, seed=i) for i, s in enumerate(((N, 96), (inner, 96), (inner, 96), (77, inner))))
    clean = orda.gated_feed_forward(x, wg, wu, wd, activation="relu")
    x[1, 7] = float("inf")
    y = orda.gated_feed_forward(x, wg, wu, wd, activation="relu")
    assert bool((y[1] == float("inf")).all())
    rest = [i for i in range(N) if i != 1]
    assert bool(y[rest].isfinite().all())
    if dtype != torch.float32:
        assert torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [4, 40, 300])
@pytest.mark.parametrize("inner", [100, 102, 129])
def test_an_infinite_gradient_of_a_row(inner, N, dtype):
    """All values positive: an infinity in the gradient from above makes dh, da, db and grad x of its row infinite."""
    x, wg, wu, wd = (positive(*s, dtype=dtype, seed=i).requires_grad_(True)
                     for i, s in enumerate(((N, 96), (inner, 96), (inner, 96), (77, inner))))
    dy = positive(N, 77, dtype=dtype, seed=9)
    clean = torch.autograd.grad(orda.gated_feed_forward(x, wg, wu, wd, activation="none"), x, dy)[0]
    dy[1, 5] = float("inf")
    got = torch.autograd.grad(orda.gated_feed_forward(x, wg, wu, wd, activation="none"), x, dy)[0]
    assert bool((got[1] == float("inf")).all())
    rest = [i for i in range(N) if i != 1]
    assert bool(got[rest].isfinite().all())
    if dtype != torch.float32:
        assert torch.equal(got[rest], clean[rest])
