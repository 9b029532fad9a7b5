"""Every engine of the projection and the feed-forward block (few-row tiles to the ring engine, K whole and in ranges) in
each product that it serves, at sizes off its tiles, against float64 on the GPU within the bounds of tests/_layers.py."""
from __future__ import annotations

import pytest
import torch

import orda_ce_kernel as orda
from tests._engine_cases import BLOCK16, BLOCK32, LINEAR16, LINEAR32
from tests._layers import ffn64, linear64

pytestmark = pytest.mark.gpu
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def inputs(shapes, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {n: (torch.randn(s, generator=g, device="cuda") * scale).to(dtype) for n, (s, scale) in shapes.items()}


def check_on_gpu(got, want):
    for name, (v, e) in want.items():
        off = (got[name].detach().double() - v).abs()
        bad = ~(off <= e)
        if bool(bad.any()):
            i = tuple(int(k) for k in bad.nonzero()[0])
            raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside the bound; first at {i}: got "
                                 f"{float(got[name][i])}, want {float(v[i])}, bound {float(e[i])}")


@pytest.mark.parametrize("size,dtype", [(s, d) for d in (BF, HF) for s in LINEAR16] + [(s, SF) for s in LINEAR32], ids=str)
def test_linear(size, dtype):
    N, K, O = size
    t = inputs({"x": ((N, K), 1.0), "w": ((O, K), K ** -0.5), "bias": ((O,), 0.5), "residual": ((N, O), 1.0), "dy": ((N, O), 1.0)},
               dtype, N + K)
    names = ("x", "w", "bias", "residual")
    leaves = [t[n].requires_grad_(True) for n in names]
    y = orda.fused_linear(*leaves, activation="silu")
    got = {"y": y, **dict(zip(names, torch.autograd.grad(y, leaves, t["dy"])))}
    check_on_gpu(got, linear64("silu", dtype, **{n: v.detach().double() for n, v in t.items()}))


@pytest.mark.parametrize("size,dtype", [(s, d) for d in (BF, HF) for s in BLOCK16] + [(s, SF) for s in BLOCK32], ids=str)
def test_block(size, dtype):
    """All gradients in one pass, then the gate's and the up weight's alone (a product of their own each)."""
    N, H, F, O = size
    t = inputs({"x": ((N, H), 1.0), "w_gate": ((F, H), H ** -0.5), "w_up": ((F, H), H ** -0.5), "w_down": ((O, F), F ** -0.5),
                "residual": ((N, O), 1.0), "dy": ((N, O), 1.0)}, dtype, N + H)
    names = ("x", "w_gate", "w_up", "w_down", "residual")
    leaves = [t[n].requires_grad_(True) for n in names]
    y = orda.gated_feed_forward(*leaves, activation="silu")
    got = {"y": y, **dict(zip(names, torch.autograd.grad(y, leaves, t["dy"], retain_graph=True)))}
    d = {n: v.detach().double() for n, v in t.items()}
    want = ffn64("silu", dtype, *[d[n] for n in names], d["dy"])
    check_on_gpu(got, want)
    for i in (1, 2):
        (alone,) = torch.autograd.grad(y, leaves[i], t["dy"], retain_graph=True)
        check_on_gpu({names[i]: alone}, {names[i]: want[names[i]]})


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("size", [(2263, 6329, 1929), (4941, 966, 5756)], ids=str)
def test_activations_on_the_ring_engine(size, dtype):
    """The forward product's epilogue of every activation, kept derivative and bias, without a residual."""
    N, K, O = size
    t = inputs({"x": ((N, K), 1.0), "w": ((O, K), K ** -0.5), "bias": ((O,), 0.5), "dy": ((N, O), 1.0)}, dtype, 3)
    bias = t["bias"].requires_grad_(True)
    d = {n: v.detach().double() for n, v in t.items()}
    for act in ("none", "relu", "gelu", "gelu_tanh", "sigmoid"):
        y = orda.fused_linear(t["x"], t["w"], bias, activation=act)
        (g,) = torch.autograd.grad(y, bias, t["dy"])
        want = linear64(act, dtype, **d)
        if act == "relu":  # (where z is within its error of the border, the derivative may be either)
            z = d["x"] @ d["w"].t() + d["bias"]
            ez = (K + 16) * 2.0 ** -24 * (d["x"].abs() @ d["w"].abs().t() + d["bias"].abs())
            v, e = want["bias"]
            want["bias"] = (v, e + (d["dy"].abs() * (z.abs() <= ez)).sum(0))
        check_on_gpu({"y": y, "bias": g}, {n: want[n] for n in ("y", "bias")})
