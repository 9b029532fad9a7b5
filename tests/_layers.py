"""Float64 definitions of the projection and the feed-forward block, and elementwise bounds of what the kernels may be off.

u is half a step of the dtype relative to the value (eps / 2); `sub` half its smallest subnormal.  Products accumulate in
fp32: gamma(K) = (K + 16) 2^-24 of the sum of magnitudes bounds any order of K additions, the exact products included (fp32
operands: each product loses 2^-23 more).  Activations: |act'| <= 1.13, |act''| <= 1; the 16-bit kernels evaluate them with
the hardware's exp2 and reciprocal, within 2^-19 (1 + |z|), fp32 with the library's functions, within 2^-20 (1 + |z|); their
derivatives within 2^-18.  A value that is rounded to the dtype and used again carries u of its magnitude on; a factor kept
for the backward pass is cut to 24 bits in 16-bit calls (2^-15 of it), exact in fp32.
"""
from __future__ import annotations

import torch

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid")
SLOPE, CURVE = 1.13, 1.0


class Unit:
    def __init__(self, dtype):
        self.u = torch.finfo(dtype).eps / 2
        self.sub = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
        self.act = 2.0 ** (-20 if dtype == torch.float32 else -19)
        self.single = dtype == torch.float32
        self.cut = 0.0 if self.single else 2.0 ** -15

    def gamma(self, n):
        return (n + 16) * 2.0 ** -24 + (2.0 ** -23 if self.single else 0.0)

    def rounded(self, v):
        return self.u * v.abs() + self.sub


def act64(name, z):
    """The activation and its derivative in float64."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name in ("sigmoid", "silu"):
        s = torch.sigmoid(z)
        return (s, s * (1 - s)) if name == "sigmoid" else (z * s, s * (1 + z * (1 - s)))
    if name == "gelu":
        p = 0.5 * torch.erfc(-z * 0.5 ** 0.5)
        return z * p, p + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    t = torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608028654 * (1 + 0.134145 * z * z)


def linear64(act, dtype, x, w, bias=None, residual=None, dy=None):
    """{name: (value, bound)} of y and, with dy, of the gradients; everything float64 on the CPU."""
    q, K = Unit(dtype), x.shape[1]
    z, s = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, s = z + bias, s + bias.abs()
    ez = q.gamma(K) * s
    f, df = act64(act, z)
    own = 0.0 if act in ("none", "relu") else q.act
    y, ey = f, SLOPE * ez + own * (1 + z.abs())
    if residual is not None:
        y, ey = y + residual, ey + 2.0 ** -23 * (f.abs() + residual.abs())
    out = {"y": (y, ey * (1 + q.u) + q.rounded(y))}
    if dy is None:
        return out
    dz = dy * df
    if act == "none":
        sums, edz = torch.zeros_like(dz), torch.zeros_like(dz)
    else:
        sums = torch.zeros_like(dz) if act == "relu" else dy.abs() * (CURVE * ez + 2.0 ** -18)
        sums = sums + q.cut * dz.abs() + 2.0 ** -24 * dz.abs()
        edz = sums + q.rounded(dz)
    out["x"] = _product(q, dz, edz, w, 0.0, w.shape[0])
    out["w"] = _product(q, dz.t(), edz.t(), x, 0.0, x.shape[0])
    if bias is not None:
        v = dz.sum(0)
        out["bias"] = (v, sums.sum(0) + q.gamma(x.shape[0]) * dz.abs().sum(0) + q.rounded(v))
    if residual is not None:
        out["residual"] = (dy, torch.zeros_like(dy))
    return out


def _product(q, a, ea, b, eb, n):
    """a @ b with errors ea, eb of its operands."""
    v = a @ b
    e = ea @ b.abs() + q.gamma(n) * (a.abs() @ b.abs())
    if not isinstance(eb, float):
        e = e + a.abs() @ eb + ea @ eb
    return v, e * (1 + q.u) + q.rounded(v)


def ffn64(act, dtype, x, wg, wu, wd, residual=None, dy=None):
    q, H, F = Unit(dtype), x.shape[1], wg.shape[0]
    a, b = x @ wg.t(), x @ wu.t()
    ea, eb = q.gamma(H) * (x.abs() @ wg.abs().t()), q.gamma(H) * (x.abs() @ wu.abs().t())
    f, df = act64(act, a)
    own = 0.0 if act in ("none", "relu") else q.act
    ef = SLOPE * ea + own * (1 + a.abs())
    h = f * b
    eh = f.abs() * eb + b.abs() * ef + ef * eb
    eh = eh + q.rounded(h)
    y, ey = _product(q, h, eh, wd.t(), 0.0, F)
    if residual is not None:
        ey = ey + 2.0 ** -23 * (y.abs() + residual.abs()) + q.rounded(residual)
        y = y + residual
    out = {"y": (y, ey)}
    if dy is None:
        return out
    dh = dy @ wd
    edh = q.gamma(wd.shape[0]) * (dy.abs() @ wd.abs())
    own1 = 0.0 if act in ("none", "relu") else 2.0 ** -18
    curve = 0.0 if act in ("none", "relu") else CURVE
    da, db = dh * b * df, dh * f
    keep = q.cut + 2.0 ** -23
    eda = (b * df).abs() * edh + (dh * df).abs() * eb + (dh * b).abs() * (curve * ea + own1) + keep * da.abs()
    edb = f.abs() * edh + dh.abs() * (SLOPE * ea + own * (1 + a.abs())) + keep * db.abs()
    eda, edb = 1.02 * eda + q.rounded(da), 1.02 * edb + q.rounded(db)  # (2%: products of errors)
    ga, gea = _product(q, da, eda, wg, 0.0, 2 * F)
    gb, geb = _product(q, db, edb, wu, 0.0, 2 * F)
    out["x"] = (ga + gb, gea + geb + q.rounded(ga + gb))
    n = x.shape[0]
    out["w_gate"] = _product(q, da.t(), eda.t(), x, 0.0, n)
    out["w_up"] = _product(q, db.t(), edb.t(), x, 0.0, n)
    out["w_down"] = _product(q, dy.t(), torch.zeros_like(dy).t(), h, eh, n)
    if residual is not None:
        out["residual"] = (dy, torch.zeros_like(dy))
    return out


def check(got, want):
    """Every output within its bound, of the right shape, with finite values only."""
    assert set(got) == set(want)
    for name, (v, e) in want.items():
        g = got[name].detach().double().cpu().reshape(v.shape)
        off = (g - v).abs()
        bad = ~(off <= e)
        if bool(bad.any()):
            i = tuple(int(k) for k in bad.nonzero()[0])
            raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside the bound; first at {i}: got "
                                 f"{float(g[i])}, want {float(v[i])}, off {float(off[i])}, bound {float(e[i])}")


def random_inputs(shapes, dtype, seed, integers=False):
    """CPU tensors in `dtype`.  `integers`: small whole numbers, whose products and sums are exact (a relu's border is then
    met exactly)."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, (shape, scale) in shapes.items():
        if integers:
            out[name] = torch.randint(-2, 3, shape, generator=g).to(dtype)
        else:
            out[name] = (torch.randn(shape, generator=g) * scale).to(dtype)
    return out
