"""Float64 definitions of a student's embedding, dropout, layer norm and attention, and elementwise bounds of what the
kernels may be off.

u is half a step of the dtype relative to the value, `sub` half its smallest subnormal (Unit, tests/_layers.py).  Sums of n
terms in fp32: gamma(n) = (n + 16) 2^-24 of the sum of magnitudes, in any order, products included.

Layer norm.  s is rounded to the dtype (error r(s) = u |s| + sub), y is computed from the unrounded s.  mean and rstd are
off by gamma(H) (mean: of mean |s|; the variance: of itself, and by the square of the mean's error), so h = (s - mean) rstd is
off by eh = rstd (e_s + e_mean + 2^-23 |s - mean|) + |h| e_rstd, with e_s = 2^-23 |s| in the forward pass and r(s) more where
the backward pass reads the rounded s.  What is made of h, g = dy w and the means follows by adding up errors of products.

Attention, per row of P, with e_z the absolute error of a score (products in fp32: gamma(D) scale |q|.|k|; the tanh: 4e-7
cap, by way of exp2 and the reciprocal; the bias: 2^-23 slope |i - j|) and one more 2^-22 (1 + |z|) for the arithmetic in
units of log2 and the hardware's exp2: P is off by P (e_z + sum P e_z + gamma(S)), and as an operand by u P (+ sub) more.
That exp2 has no subnormal results: 2^x is 0 below x = -126, so P is off by up to 2^-126 there.
The gradients: dP by gamma(D) |do|.|v|, delta by gamma(D) |do|.|o| + |do|.(error of o: u^2 |o|, it is kept in two halves, plus
that of its P), dz = P (dP - delta) (1 - t^2) by the sum of the products of the errors, and as an operand u |dz| (+ sub).
"""
from __future__ import annotations

import math

import torch

from tests._layers import Unit


def philox(block: int, site: int, seed: int):
    """The four 32-bit words of Philox4x32-10 in Python's whole numbers."""
    mask = 0xFFFFFFFF
    c = [block & mask, block >> 32, site & mask, site >> 32]
    k = [seed & mask, seed >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & mask, (a >> 32) ^ c[3] ^ k[1], a & mask]
        k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
    return c


def kept(shape, p, seed, site=0):
    """The factor of every element, float64."""
    n, drop = math.prod(shape), math.floor(p * 65536 + 0.5)
    bits = []
    for block in range((n + 7) // 8):
        for w in philox(block, site, seed):
            bits += [w & 0xFFFF, w >> 16]
    u = torch.tensor(bits[:n], dtype=torch.int64).reshape(shape)
    return (u >= drop).double() * (65536 / (65536 - drop) if drop < 65536 else 0.0)


def dropout64(dtype, x, keep, residual=None, dy=None):
    q = Unit(dtype)
    y = torch.where(keep > 0, x * keep, 0.0)
    e = 2.0 ** -23 * y.abs()
    if residual is not None:
        y, e = y + residual, e + 2.0 ** -23 * (y.abs() + residual.abs())
    out = {"y": (y, e * (1 + q.u) + q.rounded(y))}
    if dy is not None:
        dx = dy * keep
        out["x"] = (dx, 2.0 ** -22 * dx.abs() + q.rounded(dx))
        if residual is not None:
            out["residual"] = (dy, torch.zeros_like(dy))
    return out


def embedding64(dtype, out_dtype, ids, w, scale, padding_idx=None, dy=None):
    q, g = Unit(out_dtype), Unit(dtype)
    known = (ids >= 0) & (ids < w.shape[0])
    y = torch.where(known[:, None], w[ids.where(known, 0)] * scale, 0.0)
    out = {"y": (y, 2.0 ** -23 * y.abs() + q.rounded(y))}
    if dy is not None:
        take = known if padding_idx is None else known & (ids != padding_idx)
        zero = torch.zeros_like(w)
        dw = zero.index_add(0, ids[take], dy[take]) * scale
        total = zero.index_add(0, ids[take], dy[take].abs()) * abs(scale)
        n = torch.zeros(w.shape[0], dtype=torch.float64).index_add(0, ids[take], torch.ones(int(take.sum()), dtype=torch.float64))
        out["w"] = (dw, (n[:, None] + 16) * 2.0 ** -24 * total * (1 + g.u) + g.rounded(dw) * (total > 0))
    return out


def norm64(dtype, x, w, bias=None, residual=None, keep=None, eps=1e-5, dy=None, ds=None, params=None):
    """{name: (value, bound)}; params: the dtype of w and bias (default: dtype)."""
    q, H = Unit(dtype), x.shape[1]
    qp = q if params is None else Unit(params)
    gam = (H + 16) * 2.0 ** -24
    s = x if keep is None else torch.where(keep > 0, x * keep, 0.0)
    mag = s.abs()
    if residual is not None:
        mag, s = mag + residual.abs(), s + residual
    e_s = 2.0 ** -22 * mag
    mean = s.mean(1, keepdim=True)
    e_mean = gam * s.abs().mean(1, keepdim=True) + e_s.mean(1, keepdim=True)
    d = s - mean
    var = (d * d).mean(1, keepdim=True)
    e_d = e_s + e_mean + 2.0 ** -23 * (s.abs() + mean.abs())
    e_var = gam * var + (2 * d.abs() * e_d + e_d * e_d).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    # (the derivative of v^-1/2, and as much again for what is past the first order)
    e_rel = e_var / (var + eps) + 2.0 ** -21

    def normed(more):
        h = d * rstd
        e = (rstd * (e_d + more) + h.abs() * e_rel) * (1 + e_rel) + 2.0 ** -23 * h.abs()
        return h, e

    h, e_h = normed(0.0)
    y = h * w
    e_y = e_h * w.abs() + 2.0 ** -23 * y.abs()
    if bias is not None:
        y, e_y = y + bias, e_y + 2.0 ** -23 * (y.abs() + bias.abs())
    out = {"y": (y, e_y * (1 + q.u) + q.rounded(y))}
    if residual is not None:
        out["s"] = (s, e_s * (1 + q.u) + q.rounded(s))
    if dy is None:
        return out
    again = residual is None or (params is not None and params != dtype)  # (without a residual s is x, exact)
    h, e_h = normed(0.0 if again else q.rounded(s))
    g = dy * w
    mg, mgh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    e_mg = gam * g.abs().mean(1, keepdim=True) + 2.0 ** -23 * g.abs().mean(1, keepdim=True)
    e_mgh = gam * (g * h).abs().mean(1, keepdim=True) + (g.abs() * e_h).mean(1, keepdim=True) + 2.0 ** -22 * (g * h).abs().mean(1, keepdim=True)
    inner = g - mg - h * mgh
    size = g.abs() + mg.abs() + (h * mgh).abs()
    t = rstd * inner
    e_t = rstd * (e_mg + e_h * mgh.abs() + h.abs() * e_mgh + e_h * e_mgh + 2.0 ** -22 * size) * (1 + e_rel) + t.abs() * e_rel
    if ds is not None:
        t, e_t = t + ds, e_t + 2.0 ** -23 * (t.abs() + ds.abs())
    dx = t if keep is None else t * keep
    e_dx = e_t if keep is None else e_t * keep + 2.0 ** -22 * dx.abs()
    out["x"] = (dx, e_dx * (1 + q.u) + q.rounded(dx))
    if residual is not None:
        out["residual"] = (t, e_t * (1 + q.u) + q.rounded(t))
    N = x.shape[0]
    gn = (N + 16) * 2.0 ** -24
    v, e = (dy * h).sum(0), (dy.abs() * e_h).sum(0) + gn * (dy * h).abs().sum(0)
    out["w"] = (v, e * (1 + qp.u) + qp.rounded(v))
    if bias is not None:
        v = dy.sum(0)
        out["bias"] = (v, gn * dy.abs().sum(0) * (1 + qp.u) + qp.rounded(v))
    return out


def seen(B, S, causal=True, documents=None, prefix=None):
    """(B, S, S): query i sees key j."""
    i = torch.arange(S)
    m = torch.ones(B, S, S, dtype=torch.bool)
    if causal:
        m = (i[:, None] >= i[None]).expand(B, S, S).clone()
        if prefix is not None:
            for b in range(B):
                m[b, :, :max(0, int(prefix[b]))] = True
    if documents is not None:
        m &= (documents[:, :, None] == documents[:, None]) & (documents >= 0)[:, :, None]
    return m


def attention64(dtype, q, k, v, causal=True, scale=None, softcap=0.0, slopes=None, documents=None, prefix=None, dy=None,
                cap_error=None):
    """{name: (value, bound)} of (B, S, H, D) tensors; all float64.  cap_error: what a capped score may be off, of itself
    (default: 4e-7 of the cap)."""
    unit = Unit(dtype)
    B, S, H, D = q.shape
    G = H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    mask = seen(B, S, causal, documents, prefix)[:, None]
    some = mask.any(-1, keepdim=True)
    if documents is not None:
        real = (documents >= 0)[:, :, None, None]
        q, k, v = (torch.where(real, t, 0.0) for t in (q, k, v))
        dy = None if dy is None else torch.where(real, dy, 0.0)
    heads = lambda t: t.transpose(1, 2)  # noqa: E731
    shared = lambda t: heads(t).repeat_interleave(G, 1)  # noqa: E731
    qh, kh, vh = heads(q), shared(k), shared(v)
    gam = (D + 16) * 2.0 ** -24
    raw = qh @ kh.transpose(2, 3) * scale
    e_z = gam * abs(scale) * (qh.abs() @ kh.abs().transpose(2, 3))
    t = torch.zeros_like(raw)
    z = raw
    if softcap:
        t = torch.tanh(raw / softcap)
        z = softcap * t
        e_z = e_z + (4e-7 * softcap if cap_error is None else cap_error * z.abs())
    e_t = e_z / softcap if softcap else 0.0 * e_z
    if slopes is not None:
        i = torch.arange(S, dtype=torch.float64)
        bias = slopes.view(1, H, 1, 1) * (i[:, None] - i[None]).abs()
        z = z - bias
        e_z = e_z + 2.0 ** -22 * bias
    e_z = e_z + 2.0 ** -22 * (1 + z.abs())
    p = torch.where(some, torch.softmax(torch.where(some, torch.where(mask, z, -math.inf), 0.0), -1), 0.0)
    # 1.1: errors of the exponent past the first order
    e_p = 1.1 * p * (e_z + (p * e_z).sum(-1, keepdim=True) + (S + 16) * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -126 * mask
    op = lambda x, e: e * (1 + unit.u) + unit.u * x.abs() + unit.sub  # noqa: E731  (an operand, rounded)
    # the kernel holds P up to a factor between 2^-8 and 2^8 of a running maximum
    e_po = (e_p * (1 + unit.u) + unit.u * p + unit.sub) * mask
    o = p @ vh
    e_o = e_po @ vh.abs() + (S + 16) * 2.0 ** -24 * (p @ vh.abs())
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    out = {"y": (back(o), back(e_o * (1 + unit.u) + unit.rounded(o)))}
    if dy is None:
        return out
    do = heads(dy)
    dp = do @ vh.transpose(2, 3)
    e_dp = gam * (do.abs() @ vh.abs().transpose(2, 3))
    delta = (do * o).sum(-1, keepdim=True)
    e_delta = (do.abs() * (e_o + unit.u * unit.u * o.abs() + unit.sub)).sum(-1, keepdim=True) + gam * (do * o).abs().sum(-1, keepdim=True)
    f = 1 - t * t
    dz = p * (dp - delta) * f
    e_diff = e_dp + e_delta + 2.0 ** -23 * (dp.abs() + delta.abs())
    e_dz = (p + e_p) * e_diff * f + e_p * (dp - delta).abs() * f + 2.0 * (t.abs() + e_t) * e_t * p * (dp - delta).abs() + 2.0 ** -22 * dz.abs()
    e_dz = op(dz, e_dz) * mask
    gs = (S + 16) * 2.0 ** -24

    def product(a, e_a, b, n):
        v = a @ b
        return v, e_a @ b.abs() + n * (a.abs() @ b.abs())

    def grouped(x):
        return x.view(B, H // G, G, S, D).sum(2)

    v1, e1 = product(dz, e_dz, kh, gs)
    v2, e2 = product(dz.transpose(2, 3), e_dz.transpose(2, 3), qh, gs * G)
    v3, e3 = product(p.transpose(2, 3), e_po.transpose(2, 3), do, gs * G)
    for name, val, err in (("q", v1 * scale, e1 * abs(scale)), ("k", grouped(v2) * scale, grouped(e2) * abs(scale)),
                           ("v", grouped(v3), grouped(e3))):
        err = err + 2.0 ** -23 * val.abs()
        out[name] = (back(val), back(err * (1 + unit.u) + unit.rounded(val)))
    return out
