"""Capped scores at caps from where the tanh cuts to where it changes nothing, within a bound that does not contain the cap.

Below |u| = |z / cap| = 1/4 the kernels' series loses roundings of the product with scale (2^-23), of the series (2^-23) and its
next term (2^-26): less than 2^-21 of the score.  From there on tanh u = 1 - 2 / (1 + 2^a), a = 2 u / ln 2: an argument off by
2^-23 |a|, an exp2 and a reciprocal off by a step (2^-22, 2^-23) and roundings of 2^-24 are at most 4.2e-7 of absolute error at
u = 1/4, where tanh u is 0.245, and less of it behind: below 2^-19.  CAP_ERROR is twice that."""
from __future__ import annotations

import math

import pytest
import torch

import orda_ce_kernel as orda
from tests._layers import check, random_inputs
from tests._step import attention64

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
CAP_ERROR = 2.0 ** -18


def compare(B, S, H, KV, D, dtype, seed, size=1.0, **kw):
    t = random_inputs({"q": ((B, S, H, D), size), "k": ((B, S, KV, D), 1.0), "v": ((B, S, KV, D), 1.0), "dy": ((B, S, H, D), 0.3)}, dtype, seed)
    leaves = {n: t[n].cuda().requires_grad_(True) for n in "qkv"}
    y = orda.masked_attention(**leaves, **{n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in kw.items()})
    got = {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())))}
    kw = {n: v.double() if n == "slopes" else v for n, v in kw.items()}
    check(got, attention64(dtype, *(t[n].double() for n in "qkv"), dy=t["dy"].double(), cap_error=CAP_ERROR, **kw))
    return t, got


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [32, 80, 128])
@pytest.mark.parametrize("cap", [200.0, 1e3, 1e4, 1e5, 1e6, 1e7, 1e20, 1e300])
def test_large_caps(cap, D, dtype):
    compare(2, 150, 4, 2, D, dtype, D, softcap=cap)


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(slopes=torch.tensor([0.5, 0.1, 0.0, -0.02])), dict(prefix=torch.tensor([100, 0]))],
                         ids=lambda kw: "-".join(kw))
def test_large_caps_beside_other_masks(kw, D):
    compare(2, 190, 4, 2, D, BF, D + 1, softcap=1e6, **kw)
    compare(1, 40, 4, 2, D, HF, D + 2, softcap=1e6, **({**kw, "prefix": kw["prefix"][:1]} if "prefix" in kw else kw))  # (dz in two parts)


@pytest.mark.parametrize("scale", [2.0, -12.0, 60.0])
def test_scores_of_the_size_of_the_cap(scale):
    """|z / cap| on both sides of a quarter, and up to several caps."""
    t, _ = compare(1, 140, 2, 1, 64, BF, 5, size=2.0, scale=scale, softcap=150.0)
    u = (t["q"][0, :, 0].double() @ t["k"][0, :, 0].double().t() * scale / 150.0).abs()
    assert bool((u < 0.2).any()) and bool((u > 0.3).any())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_caps_that_leave_nothing_of_the_scores(dtype):
    """cap tanh(z / cap) is at most the cap: a mean of what is seen, and gradients of q and k that are zeros, or the cap's
    share of them where z is 0 to the bit."""
    t = random_inputs({n: ((1, 100, 2, 64), 1.0) for n in ("q", "k", "v")}, dtype, 6)
    want = orda.masked_attention(*(t[n].cuda() for n in "qkv"), scale=0.0)
    for cap in (1e-300, 1e-30, 1e-12):
        leaves = [t[n].cuda().requires_grad_(True) for n in "qkv"]
        y = orda.masked_attention(*leaves, softcap=cap)
        assert float((y - want).abs().max()) <= float(want.abs().max()) * 2 * torch.finfo(dtype).eps
        assert all(torch.isfinite(g).all() for g in torch.autograd.grad(y.float().sum(), leaves))


def test_a_cap_past_any_score_is_none():
    t = random_inputs({n: ((1, 300, 2, 64), 1.0) for n in ("q", "k", "v")}, HF, 7)
    q, k, v = (t[n].cuda() for n in "qkv")
    none, far = orda.masked_attention(q, k, v).double(), orda.masked_attention(q, k, v, softcap=1e30).double()
    assert float((none - far).norm()) <= 2 * torch.finfo(HF).eps * float(none.norm())
    assert math.isfinite(float(far.sum()))
