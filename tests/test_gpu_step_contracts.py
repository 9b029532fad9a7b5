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


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("dtype", [BF, torch.float16])
@pytest.mark.parametrize("kw", [dict(scale=0.0), dict(scale=1e-20), dict(softcap=3.0), dict()], ids=lambda kw: "-".join(kw) or "plain")
def test_slopes_past_the_range_of_fp32(kw, dtype, D):
    """Slopes of any finite size: a query sees itself alone, with a negative one the first key alone; o is that key's v and
    no score has a gradient to speak of.  (Of the negative ones the backward pass has P = 2^(z - L) from L in fp32, and z is up to 2^22
    there, which fp32 holds to a quarter: dv is off by up to 2^(1/4).)"""
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(1, 150, h, D, generator=g).to(dtype).cuda().requires_grad_(True) for h in (4, 2, 2))
    slopes = torch.tensor([1e16, 3e38, -1e16, -3e38], device="cuda")
    y = orda.masked_attention(q, k, v, slopes=slopes, **kw)
    assert torch.equal(y[:, :, 0], v[:, :, 0]) and torch.equal(y[:, :, 1], v[:, :, 0])
    assert torch.equal(y[:, :, 2], v[:, :1, 1].expand(1, 150, D)) and torch.equal(y[:, :, 3], v[:, :1, 1].expand(1, 150, D))
    dq, dk, dv = torch.autograd.grad(y, (q, k, v), torch.ones_like(y))
    assert not dq[:, :, :2].any() and not dk[:, :, 0].any()
    # (the key's own P, 2^(up to 1/4), is rounded as an operand and divided out by a reciprocal: 2^-24 of o are left in delta,
    # 2^-23 |v| of it with a score's rounding, times P <= 1.2, scale and k or, over 300 queries, q)
    off = abs(kw.get("scale", D ** -0.5)) * 1.2 * 2.0 ** -23 * float(v.detach()[0, 0, 1].float().abs().sum())
    assert float(dq.float().abs().max()) <= off * float(k.detach().float().abs().max())
    assert float(dk.float().abs().max()) <= off * 300 * float(q.detach().float().abs().max())
    assert torch.equal(dv[:, :, 0], torch.full_like(dv[:, :, 0], 2.0)) and not dv[:, 1:, 1].any()
    assert bool((dv[:, 0, 1] >= 300 / 1.2).all()) and bool((dv[:, 0, 1] <= 300 * 1.2).all())


@pytest.mark.parametrize("dtype", [BF, torch.float16])
def test_steep_slopes_over_long_rows(dtype):
    """Far keys' scores of -1e5 to -2e9 before a query's own come last: it sees itself alone, to the bit."""
    g = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(1, 3000, h, 64, generator=g).to(dtype).cuda().requires_grad_(True) for h in (4, 1, 1))
    y = orda.masked_attention(q, k, v, slopes=torch.tensor([200.0, 1e4, 3e5, 7e5], device="cuda"))
    assert torch.equal(y, v.expand_as(y))
    dq, dk, dv = torch.autograd.grad(y, (q, k, v), torch.ones_like(y))
    assert not dq.any() and not dk.any() and torch.equal(dv, torch.full_like(dv, 4.0))
