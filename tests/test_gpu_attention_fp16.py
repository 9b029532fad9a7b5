"""Gradients of fp16 attention where probabilities and dz lie among fp16's subnormals, or dz past its largest value: long rows,
small and large gradients from above, and both in one call.

The bound, per gradient, of the error's norm: what half steps (u = 2^-11) of the operands P and dz and of the result leave.
Roundings of different elements are independent, so those of a sum of products a b add up as sqrt(sum (u a b)^2); the factor
between u and the standard deviation of a rounding (more than 2: it is even between -u and u at most) is left as reserve.
delta = do o is off by what P's roundings leave of it, sqrt(sum (u P do v)^2), and dz by P times that, for all keys of a row
alike.  The three parts are added, which is more than their root of squares.  A result has in fp16 steps of 2^-24 below 2^-14:
half a step more for each element.  fp32 sums are 2^-17 of their absolute sums off at most, below u's part."""
from __future__ import annotations

import math

import pytest
import torch

import orda_ce_kernel as orda

pytestmark = pytest.mark.gpu
HF = torch.float16
U, SUB = torch.finfo(HF).eps / 2, 2.0 ** -25


def inputs(S, H, KV, D, seed=1, peak=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = {n: torch.randn(1, S, h, D, generator=g, device="cuda") for n, h in (("q", H), ("k", KV), ("v", KV), ("dy", H))}
    t["q"] *= peak
    return t


def run(t, **kw):
    leaves = [t[n].to(HF).requires_grad_(True) for n in "qkv"]
    y = orda.masked_attention(*leaves, **kw)
    return dict(zip("qkv", torch.autograd.grad(y, leaves, t["dy"].to(HF))))


def compare(t, causal=True, softcap=0.0, rows=None):
    """rows: the queries whose dq is compared by itself, each row against its own bound."""
    got = run(t, causal=causal, softcap=softcap)
    S, H, D = t["q"].shape[1:]
    KV, scale, step = t["k"].shape[2], D ** -0.5, 2048
    q, k, v, dy = (t[n][0].to(HF).double() for n in ("q", "k", "v", "dy"))
    at = torch.arange(S, device="cuda")
    want = {n: torch.zeros_like(x) for n, x in (("q", q), ("k", k), ("v", v))}
    first, second = ({n: torch.zeros_like(x) for n, x in want.items()} for _ in range(2))  # (squares: of the operand, of delta)
    for h in range(H):
        c, s = h * KV // H, scale * scale
        K, V = k[:, c], v[:, c]
        for i in range(0, S, step):
            Q, g = q[i:i + step, h], dy[i:i + step, h]
            z, f = Q @ K.t() * scale, 1.0
            if softcap:
                th = torch.tanh(z / softcap)
                z, f = softcap * th, 1 - th * th
            if causal:
                z = z.masked_fill(at[i:i + step, None] < at, -math.inf)
            p = torch.softmax(z, -1)
            dp = g @ V.t()
            delta = (p * dp).sum(-1, keepdim=True)
            off = U * U * (p * p * dp * dp).sum(-1, keepdim=True)
            dz = p * (dp - delta) * f
            want["q"][i:i + step, h] = scale * dz @ K
            first["q"][i:i + step, h] = s * U * U * (dz * dz) @ (K * K)
            second["q"][i:i + step, h] = s * off * ((p * f) @ K) ** 2
            want["k"][:, c] += scale * dz.t() @ Q
            first["k"][:, c] += s * U * U * (dz * dz).t() @ (Q * Q)
            second["k"][:, c] += s * (p * p * f * f * off).t() @ (Q * Q)
            want["v"][:, c] += p.t() @ g
            first["v"][:, c] += U * U * (p * p).t() @ (g * g)
    for n in want:
        # (a sum past fp16's largest value, 65504, is an infinity: such are looked at by themselves)
        large = want[n].abs() > 65000
        assert bool((got[n][0].abs()[large] > 64000).all()) and bool(torch.isfinite(got[n][0][~large]).all()), n
        e, w = torch.where(large, 0.0, got[n][0].double() - want[n]), want[n]
        if n == "q" and rows is not None:
            e, w, a, b = (x[rows] for x in (e, w, first[n], second[n]))
            dims = (1, 2)
        else:
            a, b, dims = first[n], second[n], (0, 1, 2)
        off = e.square().sum(dims).sqrt()
        bound = a.sum(dims).sqrt() + b.sum(dims).sqrt() + U * w.square().sum(dims).sqrt() + SUB * math.prod(w.shape[i] for i in dims) ** 0.5
        assert bool((off <= bound).all()), (n, float((off / bound).max()), float(off.max()), float(w.norm()))
    return got


@pytest.mark.parametrize("dy", [1.0, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("S", [300, 2048, 4096, 16384])
def test_small_gradients_from_above(S, dy):
    t = inputs(S, 1, 1, 64, S)
    t["dy"] *= dy
    compare(t, causal=S == 2048)


@pytest.mark.parametrize("D,H,KV", [(24, 4, 1), (80, 2, 1), (96, 4, 4), (128, 2, 1)])
@pytest.mark.parametrize("dy", [1e-2, 1e-4])
def test_small_gradients_of_every_width(dy, D, H, KV):
    """Heads of a key one after the other and in parts."""
    t = inputs(2500, H, KV, D, D)
    t["dy"] *= dy
    compare(t, causal=False)
    compare(t, softcap=5.0)


@pytest.mark.parametrize("S", [40, 64, 300])
@pytest.mark.parametrize("dy", [1e2, 1e3, 2e4])
def test_large_gradients_from_above(dy, S):
    """dz past fp16's 65504 before it meets keys and queries that are small."""
    t = inputs(S, 2, 1, 64, S, peak=3.0)
    t["dy"] = (t["dy"] * dy).clamp(-6e4, 6e4)
    t["k"], t["q"], t["v"] = t["k"] * 0.02, t["q"] * 0.02, t["v"] * 0.2
    compare(t)
    for D in (80, 128):
        u = inputs(S, 2, 2, D, S, peak=3.0)
        u["dy"] = (u["dy"] * dy).clamp(-6e4, 6e4)
        u["k"], u["q"], u["v"] = u["k"] * 0.02, u["q"] * 0.02, u["v"] * 0.2
        compare(u)


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_gradients_from_above_of_many_sizes(order, D):
    """From 1e-4 to 1e3 over the queries: sums that go down by powers of two on the way, and each query's dq by itself."""
    S = 1000
    size = torch.logspace(-4, 3, S, device="cuda")
    if order == "down":
        size = size.flip(0)
    if order == "mixed":
        size = size[torch.randperm(S, generator=torch.Generator().manual_seed(2)).cuda()]
    t = inputs(S, 2, 1, D, 7)
    t["dy"] = t["dy"] * size[:, None, None]
    t["v"] = t["v"] * 0.3
    t["k"] = t["k"] * 0.3
    compare(t, causal=False, rows=slice(None))
    compare(t, rows=slice(64, None))  # (the first rows see few keys: no sum of roundings to speak of)


def test_values_of_many_sizes_along_the_keys():
    """dz grows along a query's keys, by rows of v of 1e-3 to 1e3."""
    t = inputs(1500, 2, 2, 64, 8)
    t["v"] = t["v"] * torch.logspace(-3, 3, 1500, device="cuda")[:, None, None]
    t["dy"] *= 1e-3
    compare(t)
    t["v"] = t["v"].flip(1)
    compare(t, causal=False)


def test_zero_gradients_from_above():
    t = inputs(500, 2, 1, 64, 9)
    t["dy"].zero_()
    assert not any(g.any() for g in run(t).values())
    t["dy"][0, 400] = 1.0
    got = run(t)
    assert not got["q"][0, :400].any() and got["q"][0, 400].any() and not got["q"][0, 401:].any() and not got["v"][0, 401:].any()


def test_long_tails_of_small_probabilities():
    """Half of the output comes from 60000 keys whose probabilities are 2^-17 of the largest each.  The largest key's scores
    are 2^17's logarithm above the others': y is their mean with it, to half a step of P (2^-11 of each part, of independent
    signs) and of y."""
    S, D = 60001, 64
    q = torch.zeros(1, S, 1, D, device="cuda", dtype=HF)
    k, v = torch.zeros_like(q), torch.full_like(q, 1.0)
    q[:, :, :, 0] = 1.0
    k[0, 0, 0, 0] = 17 * math.log(2)
    v[0, 0] = -1.0
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    y = orda.masked_attention(*leaves, scale=1.0, causal=False)
    top = math.exp(float(k.detach()[0, 0, 0, 0].double()))
    want = (S - 1 - top) / (S - 1 + top)
    share = (S - 1) / (S - 1 + top)
    assert abs(float(y.detach()[0, 0, 0, 0]) - want) <= 2 * U * (share + abs(want) + (1 - share))
    (dv,) = torch.autograd.grad(y, v, torch.full_like(y, 2.0 ** -6))
    assert abs(float(dv[0, 5, 0, 0]) - S * 2.0 ** -6 / (S - 1 + top)) <= 2 * U * S * 2.0 ** -6 / (S - 1 + top)
