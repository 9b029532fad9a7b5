"""The token embedding, dropout and the layer norm on the kernels, against float64 within the bounds of tests/_step.py: every
width that a kernel is chosen by, odd sizes, strides, dtypes, rows that are special."""
from __future__ import annotations

import math

import pytest
import torch

import orda_ce_kernel as orda
from tests._layers import Unit, check, random_inputs
from tests._step import dropout64, embedding64, kept, norm64

pytestmark = pytest.mark.gpu
BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def wide(t):
    return {n: v.double() if v.is_floating_point() else v for n, v in t.items()}


# ------------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("shape,p,seed,site", [((1,), 0.5, 0, 0), ((7,), 0.5, 1, 0), ((3, 5, 9), 0.1, 2**64 - 1, 2**63), ((40, 104), 0.9, 3, 1),
                                               ((2, 1000), 0.0, 4, 0), ((5, 33), 1.0, 5, 0), ((4, 16), 2.0**-17, 6, 0)])
def test_dropout(shape, p, seed, site, dtype):
    t = random_inputs({n: (shape, 1.0) for n in ("x", "residual", "dy")}, dtype, 1)
    for with_residual in (False, True):
        leaves = {n: t[n].cuda().requires_grad_(True) for n in (("x", "residual") if with_residual else ("x",))}
        y = orda.counter_dropout(leaves["x"], p, leaves.get("residual"), seed=seed, site=site)
        got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())))
        d = wide(t)
        check({"y": y, **got}, dropout64(dtype, d["x"], kept(shape, p, seed, site), d["residual"] if with_residual else None, d["dy"]))


@pytest.mark.parametrize("dtype", [BF, F])
def test_dropout_does_not_depend_on_strides(dtype):
    """Transposed, sliced, expanded and unaligned tensors have the mask of their elements' indices."""
    x = torch.randn(37, 50, device="cuda").to(dtype)
    want = orda.counter_dropout(x, 0.4, seed=9)
    pitched = torch.zeros(37, 61, dtype=dtype, device="cuda")[:, 3:53]
    pitched.copy_(x)
    odd = torch.zeros(37 * 50 + 1, dtype=dtype, device="cuda")[1:].view(37, 50).copy_(x)
    for same in (pitched, x.t().contiguous().t(), odd):
        assert torch.equal(orda.counter_dropout(same, 0.4, seed=9), want)
        assert torch.equal(orda.counter_dropout(x, 0.4, same, seed=9), orda.counter_dropout(x, 0.4, x, seed=9))
    row = x[:1].expand(37, 50)
    assert torch.equal(orda.counter_dropout(row, 0.4, seed=9), orda.counter_dropout(row.contiguous(), 0.4, seed=9))


def test_dropped_infinities_leave_nothing():
    x = torch.full((8, 64), math.inf, device="cuda")
    x[:, ::3] = math.nan
    keep = kept((8, 64), 0.5, 3).cuda()
    y = orda.counter_dropout(x, 0.5, seed=3)
    assert torch.equal(y == 0, keep == 0)
    assert not orda.counter_dropout(x, 1.0, seed=3).any()


def test_dropout_past_32_bits():
    """More than 2^32 elements: the counter's high word, and the last ones against their own."""
    n = (1 << 32) + 4097
    x = torch.ones(n, dtype=BF, device="cuda")
    y = orda.counter_dropout(x, 0.5, seed=11)
    from tests._step import philox
    for first in (0, (1 << 32) - 16, 1 << 32, n // 8 * 8 - 16):
        bits = [b for k in range(2) for w in philox(first // 8 + k, 0, 11) for b in (w & 0xFFFF, w >> 16)]
        assert y[first:first + 16].tolist() == [2.0 if b >= 32768 else 0.0 for b in bits]
    share = float(y.count_nonzero()) / n
    assert abs(share - 0.5) < 5 * 0.5 / math.sqrt(n)  # (five standard deviations; the seed is fixed)


# ------------------------------------------------------------------- layer norm
WIDTHS = [1, 7, 8, 63, 64, 65, 512, 513, 777, 1024, 1111, 2048, 2056, 4096, 4097, 5120, 8192, 8200, 16384]


def norm_case(N, H, dtype, seed, params=None):
    t = random_inputs({"x": ((N, H), 1.0), "residual": ((N, H), 1.0), "dy": ((N, H), 0.1), "ds": ((N, H), 0.1)}, dtype, seed)
    p = random_inputs({"w": ((H,), 0.3), "bias": ((H,), 0.3)}, params or dtype, seed + 1)
    t["residual"] = t["residual"] + 0.5
    t["w"], t["bias"] = p["w"] + 1, p["bias"]
    return t


def run_norm(t, p=0.0, seed=5, **kw):
    leaves = {n: t[n].cuda().requires_grad_(True) for n in ("x", "residual", "w", "bias") if n in t}
    got = orda.layer_norm(leaves["x"], leaves["w"], leaves.get("bias"), leaves.get("residual"), p=p, seed=seed, **kw)
    out = dict(zip(("y", "s"), got if isinstance(got, tuple) else (got,)))
    above = [t[n].cuda() for n in (("dy", "ds") if "residual" in t else ("dy",))]
    return {**{n: v.detach() for n, v in out.items()}, **dict(zip(leaves, torch.autograd.grad(list(out.values()), list(leaves.values()), above)))}


def want_norm(t, dtype, p=0.0, seed=5, **kw):
    d = wide(t)
    keep = kept(tuple(t["x"].shape), p, seed) if p else None
    return norm64(dtype, d["x"], d["w"], d.get("bias"), d.get("residual"), keep, dy=d["dy"], ds=d["ds"] if "residual" in t else None,
                  params=t["w"].dtype, **kw)


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("H", WIDTHS)
def test_norm(H, dtype):
    t = norm_case(5, H, dtype, 10 + H)
    del t["residual"]
    check(run_norm(t), want_norm(t, dtype))


@pytest.mark.parametrize("dtype,params", [(BF, None), (HF, None), (F, None), (HF, F), (BF, F)])
@pytest.mark.parametrize("N,H", [(1, 24), (37, 40), (3, 777), (70, 1111), (5, 2048), (3, 4096), (2, 5121), (3, 8200)])
def test_norm_with_dropout_and_residual(N, H, dtype, params):
    t = norm_case(N, H, dtype, 3 * H + N, params)
    check(run_norm(t, 0.3), want_norm(t, dtype, 0.3))
    del t["bias"]
    check(run_norm(t), want_norm(t, dtype))


@pytest.mark.parametrize("N,H", [(3000, 8), (1500, 96), (700, 1000), (1100, 1500), (600, 2560), (300, 8200)])
def test_norm_of_more_rows_than_workgroups(N, H):
    """Each workgroup walks several rows and adds up its share of dw and db."""
    t = norm_case(N, H, BF, N + H)
    check(run_norm(t, 0.0), want_norm(t, BF))
    t = norm_case(N, H, HF, N, F)
    check(run_norm(t, 0.1), want_norm(t, HF, 0.1))


def test_norm_of_strided_and_unaligned_rows():
    t = norm_case(9, 100, BF, 4)
    plain = run_norm(t, 0.2)
    big = torch.zeros(9, 230, dtype=BF)
    big[:, 1:101], big[:, 121:221] = t["x"], t["residual"]
    big = big.cuda()
    leaves = {"x": big[:, 1:101].detach().requires_grad_(True), "residual": big[:, 121:221].detach().requires_grad_(True),
              "w": t["w"].cuda().repeat_interleave(2)[::2].requires_grad_(True), "bias": torch.cat([t["bias"][:1], t["bias"]])[1:].cuda().requires_grad_(True)}
    leaves = {n: v.detach().requires_grad_(True) for n, v in leaves.items()}
    y, s = orda.layer_norm(leaves["x"], leaves["w"], leaves["bias"], leaves["residual"], p=0.2, seed=5)
    above = [torch.zeros(9, 300, dtype=BF, device="cuda")[:, a:a + 100] for a in (3, 150)]
    for a, n in zip(above, ("dy", "ds")):
        a.copy_(t[n])
    got = dict(zip(leaves, torch.autograd.grad((y, s), list(leaves.values()), above)))
    for n, v in {"y": y, "s": s, **got}.items():
        assert torch.equal(v, plain[n]), n
    x3 = t["x"].cuda().view(3, 3, 100).transpose(0, 1)
    assert torch.equal(orda.layer_norm(x3, leaves["w"]), orda.layer_norm(x3.contiguous().view(9, 100), leaves["w"]).view(3, 3, 100))


def test_norm_gradients_one_at_a_time():
    """Any subset of gradients gives the bits of all of them; an unused y or s counts as a zero gradient."""
    t = norm_case(40, 264, BF, 6)
    every = run_norm(t, 0.2)
    for want in ("x", "residual", "w", "bias"):
        leaves = {n: t[n].cuda().requires_grad_(n == want) for n in ("x", "residual", "w", "bias")}
        y, s = orda.layer_norm(leaves["x"], leaves["w"], leaves["bias"], leaves["residual"], p=0.2, seed=5)
        (g,) = torch.autograd.grad((y, s), leaves[want], (t["dy"].cuda(), t["ds"].cuda()))
        assert torch.equal(g, every[want]), want
    for used, zero in (("dy", "ds"), ("ds", "dy")):
        leaves = {n: t[n].cuda().requires_grad_(True) for n in ("x", "residual", "w", "bias")}
        out = dict(zip(("dy", "ds"), orda.layer_norm(leaves["x"], leaves["w"], leaves["bias"], leaves["residual"], p=0.2, seed=5)))
        got = torch.autograd.grad(out[used], list(leaves.values()), t[used].cuda())
        same = run_norm({**t, zero: torch.zeros_like(t[zero])}, 0.2)
        assert all(torch.equal(g, same[n]) for n, g in zip(leaves, got))


def test_norm_of_special_rows():
    """A constant row (variance 0), one far from zero, and an infinity, which stays in its own row."""
    x = torch.randn(6, 200, device="cuda")
    x[0] = 3.0
    x[1] = x[1] * 1e-3 + 1e4  # (fp32: 1e4 + 1e-3 keeps 1e-3 to 1e-3 of itself)
    x[2, 5] = math.inf
    w = torch.ones(200, device="cuda")
    y = orda.layer_norm(x, w)
    assert torch.equal(y[0], torch.zeros(200, device="cuda"))
    assert torch.isnan(y[2]).any() and torch.isfinite(y[3:]).all()
    check({"y": y[1:2]}, {"y": norm64(F, x[1:2].cpu().double(), w.cpu().double())["y"]})
    zero = torch.zeros(2, 16, device="cuda", requires_grad=True)
    y = orda.layer_norm(zero, torch.ones(16, device="cuda"), eps=0.0)
    assert torch.isnan(y).all()  # (0 / 0, as the formula has it)


def test_norm_past_32_bits():
    """More than 2^32 elements: rows at both ends against their own results, dw of whole rows."""
    H, N = 4096, (1 << 20) + 3
    x = torch.randn(1 << 12, H, device="cuda").to(BF).repeat(257, 1)[:N].requires_grad_(True)
    w = torch.ones(H, device="cuda", dtype=BF, requires_grad=True)
    y = orda.layer_norm(x, w)
    some = torch.cat([x[:5].detach(), x[-5:].detach()]).requires_grad_(True)
    z = orda.layer_norm(some, w)
    assert torch.equal(torch.cat([y[:5], y[-5:]]).detach(), z.detach())
    dy = torch.zeros(N, H, device="cuda", dtype=BF)
    dy[:5], dy[-5:] = 1.0, 0.5
    dy[:, ::2] *= -1
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    hx, hw = torch.autograd.grad(z, (some, w), torch.cat([dy[:5], dy[-5:]]))
    assert torch.equal(torch.cat([gx[:5], gx[-5:]]), hx) and not gx[5:-5].any()
    assert float((gw.double() - hw.double()).abs().max()) <= 2 * Unit(BF).u * float(hw.abs().max()) + 1e-6


# ------------------------------------------------------------------- embedding
def embed_case(N, V, H, dtype, seed, out=None, spread=1.0, bad=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(N, generator=g) ** spread * V).long().clamp(max=V - 1)
    if bad:
        off = torch.rand(N, generator=g) < bad
        ids[off] = torch.tensor([-100, V, 2**40, -(2**40)])[torch.randint(4, (int(off.sum()),), generator=g)]
    t = random_inputs({"w": ((V, H), 1.0)}, dtype, seed)
    t["dy"] = random_inputs({"dy": ((N, H), 0.5)}, out or dtype, seed + 1)["dy"]
    return {"ids": ids, **t}


def run_embed(t, scale=1.0, padding_idx=None):
    w = t["w"].cuda().requires_grad_(True)
    y = orda.token_embedding(t["ids"].cuda(), w, scale=scale, padding_idx=padding_idx)
    (g,) = torch.autograd.grad(y, w, t["dy"].cuda())
    return {"y": y.detach(), "w": g}


@pytest.mark.parametrize("dtype", [BF, HF, F])
@pytest.mark.parametrize("N,V,H", [(1, 1, 1), (3, 5, 8), (64, 2, 33), (100, 255, 64), (257, 256, 40), (500, 65536, 24), (4095, 300, 17), (4096, 7, 8),
                                   (4097, 1000, 16), (9000, 70000, 9), (300, 50, 1111), (70, 33, 4096)])
def test_embedding(N, V, H, dtype):
    t = embed_case(N, V, H, dtype, N + V + H, spread=3.0, bad=0.1)
    d = wide(t)
    check(run_embed(t, 1.75, V // 3), embedding64(dtype, dtype, t["ids"], d["w"], 1.75, V // 3, d["dy"]))


@pytest.mark.parametrize("N", [1, 31, 32, 33, 1000, 5000, 70000])
@pytest.mark.parametrize("H", [8, 600])
def test_one_token_fills_the_batch(N, H):
    """One run over all chunks, and two that meet in a chunk."""
    if N * H > 5_000_000:
        H = 40
    for ids in (torch.full((N,), 2), torch.arange(N) * 2 // N + 1):
        t = {**embed_case(N, 4, H, F, N + H), "ids": ids}
        d = wide(t)
        check(run_embed(t), embedding64(F, F, ids, d["w"], 1.0, None, d["dy"]))


def test_every_token_once_and_none():
    t = {**embed_case(5000, 5000, 16, F, 3), "ids": torch.randperm(5000, generator=torch.Generator().manual_seed(1))}
    got = run_embed(t, 0.5)
    assert torch.equal(got["w"].cpu()[t["ids"]], t["dy"] * 0.5) and torch.equal(got["y"].cpu(), t["w"][t["ids"]] * 0.5)
    got = run_embed({**t, "ids": torch.full((5000,), -1)})
    assert not got["w"].any() and not got["y"].any()


def test_long_batches_are_merged_in_rounds():
    """Past 16 segments of 4096 tokens; small whole numbers, exact sums, so that a lost or doubled entry shows."""
    N, V = 16 * 4096 * 3 + 5, 977
    g = torch.Generator(device="cuda").manual_seed(2)
    ids = torch.randint(-3, V + 3, (N,), generator=g, device="cuda")
    dy = torch.randint(-2, 3, (N, 8), generator=g, device="cuda").float()
    w = torch.zeros(V, 8, device="cuda", requires_grad=True)
    (got,) = torch.autograd.grad(orda.token_embedding(ids, w), w, dy)
    ok = (ids >= 0) & (ids < V)
    want = torch.zeros(V, 8, device="cuda", dtype=torch.float64).index_add_(0, ids[ok], dy[ok].double())
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("N,V,H,dtype", [(100, 40000, 4099, BF), (5000, 70001, 4096, BF), (4200, 150000, 1001, HF), (9, 12_000_000, 8, F), (70000, 90000, 1032, F)])
def test_rows_that_no_token_names_are_zeros(N, V, H, dtype):
    """Gradients of more bytes than are filled beside the sort and the merge, over memory that held NaN; whole numbers, exact sums."""
    g = torch.Generator(device="cuda").manual_seed(N)
    ids = torch.randint(-2, V + 2, (N,), generator=g, device="cuda")
    ids[::3] = V - 1 - ids[::3].abs() % 7
    ids[1::5] = 70
    dy = torch.randint(-1, 2, (N, H), generator=g, device="cuda").to(dtype)
    w = torch.zeros(V, H, dtype=dtype, device="cuda", requires_grad=True)
    y = orda.token_embedding(ids, w, padding_idx=V // 2)
    held = torch.full((V, H), float("nan"), dtype=dtype, device="cuda")
    del held
    (got,) = torch.autograd.grad(y, w, dy)
    ok = (ids >= 0) & (ids < V) & (ids != V // 2)
    rows, at = ids[ok].unique(return_inverse=True)
    want = torch.zeros(len(rows), H, device="cuda", dtype=torch.float64).index_add_(0, at, dy[ok].double())
    assert torch.equal(got[rows].double(), want.to(dtype).double())
    got[rows] = 0
    assert not got.any()


def test_embedding_gradients_are_the_same_in_every_run():
    t = embed_case(6000, 200, 72, HF, 5, spread=4.0)
    first = run_embed(t)
    for _ in range(3):
        again = run_embed(t)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_embedding_dtypes_strides_and_shapes():
    """int32 ids of any shape and stride, pitched weights, autocast (fp32 weight and gradient, 16-bit rows), pitched dy."""
    t = embed_case(60, 90, 40, F, 8, out=BF)
    ids = t["ids"].int().cuda()
    w = torch.zeros(90, 57, device="cuda")[:, 5:45].copy_(t["w"]).requires_grad_(True)
    pitched = torch.zeros(60, 99, dtype=BF, device="cuda")[:, 3:43].copy_(t["dy"])
    with torch.autocast("cuda", dtype=BF):
        y = orda.token_embedding(ids.view(5, 12), w, scale=3.0)
    assert y.dtype == BF and y.shape == (5, 12, 40)
    (g,) = torch.autograd.grad(y.view(60, 40), w, pitched)
    assert g.dtype == F
    d = wide(t)
    check({"y": y, "w": g}, embedding64(F, BF, t["ids"], d["w"], 3.0, None, d["dy"]))
    assert torch.equal(orda.token_embedding(ids.view(5, 12).t(), w), orda.token_embedding(ids.view(5, 12).t().contiguous(), w))
    with torch.autocast("cuda", dtype=HF):
        assert orda.token_embedding(ids[:0], w).dtype == HF


def test_embedding_past_32_bits():
    """A weight, a gradient and rows of more than 2^32 bytes and 2^31 elements each."""
    V, H = (1 << 20) + 5, 2056
    w = torch.zeros(V, H, dtype=BF, device="cuda")
    w[::4096] = 1.0
    w[-1] = 2.0
    w.requires_grad_(True)
    N = (1 << 20) + 9
    ids = torch.full((N,), 5, device="cuda")
    ids[-3:] = V - 1
    ids[:4096:2] = 4096
    y = orda.token_embedding(ids, w)
    assert bool((y[-3:] == 2).all()) and bool((y[:4096:2] == 1).all()) and not y[1:4096:2].any()
    dy = torch.zeros(N, H, dtype=BF, device="cuda")
    dy[-3:] = 1.0
    dy[:4096:2] = 0.5
    dy[-4] = 3.0
    (g,) = torch.autograd.grad(y, w, dy)
    assert bool((g[-1] == 3).all()) and bool((g[4096] == 1024).all()) and bool((g[5] == 3).all())
    assert int(g.count_nonzero()) == 3 * H
