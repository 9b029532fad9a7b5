"""Masked attention on the kernels, against float64 within the bounds of tests/_step.py: lengths around the tiles, every
mask, head layouts, strides, special rows."""
from __future__ import annotations

import math

import pytest
import torch

import orda_ce_kernel as orda
from tests._layers import check, random_inputs
from tests._step import attention64

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def case(B, S, H, KV, D, dtype, seed, scale=1.0):
    return random_inputs({"q": ((B, S, H, D), scale), "k": ((B, S, KV, D), scale), "v": ((B, S, KV, D), 1.0), "dy": ((B, S, H, D), 0.3)}, dtype, seed)


def on_gpu(kw):
    return {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in kw.items()}


def run(t, **kw):
    leaves = {n: t[n].cuda().requires_grad_(True) for n in ("q", "k", "v")}
    y = orda.masked_attention(**leaves, **on_gpu(kw))
    return {"y": y.detach(), **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())))}


def want(t, dtype, **kw):
    d = {n: v.double() for n, v in t.items()}
    kw = {n: v.double() if n == "slopes" else v for n, v in kw.items()}
    return attention64(dtype, d["q"], d["k"], d["v"], dy=d["dy"], **kw)


def compare(t, dtype, **kw):
    with torch.no_grad():
        still = orda.masked_attention(*(t[n].cuda() for n in ("q", "k", "v")), **on_gpu(kw))
    got = run(t, **kw)
    assert torch.equal(still, got["y"])
    check(got, want(t, dtype, **kw))
    return got


def documents(B, S, seed, pad=True):
    """Runs of numbers, some again later, some of padding."""
    g = torch.Generator().manual_seed(seed)
    out = torch.empty(B, S, dtype=torch.int32)
    for b in range(B):
        at = 0
        while at < S:
            n = int(torch.randint(1, max(2, S // 3), (), generator=g))
            out[b, at:at + n] = int(torch.randint(-1 if pad else 0, 4, (), generator=g))
            at += n
    return out


SLOPES = lambda H: torch.exp2(-torch.arange(1, H + 1, dtype=torch.float32))  # noqa: E731


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S", [1, 2, 31, 33, 63, 64, 65, 127, 128, 129, 200, 300])
def test_lengths(S, causal, dtype):
    compare(case(2, S, 2, 1, 64, dtype, S), dtype, causal=causal)


@pytest.mark.parametrize("D", [1, 3, 8, 12, 16, 40, 63, 64, 65, 72, 80, 100, 120, 127, 128])
def test_head_dims(D):
    compare(case(1, 150, 3, 3, D, HF, D), HF, causal=True)


@pytest.mark.parametrize("H,KV", [(1, 1), (6, 2), (8, 1), (5, 5)])
@pytest.mark.parametrize("D", [64, 128])
def test_shared_heads(H, KV, D):
    compare(case(2, 190, H, KV, D, BF, H + D), BF)


@pytest.mark.parametrize("B,S,H,KV,D", [
    (32, 130, 16, 8, 40),   # 512 tiles of keys: a workgroup takes all heads of its keys
    (16, 130, 24, 8, 64),   # 256: two take three heads, one of them one
    (16, 130, 32, 8, 96),   # 256: two take two heads each
    (16, 130, 16, 8, 128),  # 256: two take one each
    (18, 150, 20, 4, 112),  # 144: four for five heads, by twos: three
])
def test_parts_of_shared_heads(B, S, H, KV, D):
    """Heads that share keys one after the other in a workgroup, each in one of its own, and between the two."""
    compare(case(B, S, H, KV, D, BF, H + D), BF, documents=documents(B, S, D), prefix=torch.arange(B, dtype=torch.int32) * 9)


@pytest.mark.parametrize("D", [65, 68, 81, 88, 95, 96, 97, 104])
def test_head_dims_around_96(D):
    compare(case(2, 140, 4, 2, D, BF, D), BF, causal=False, softcap=3.0)


@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("kw", [
    dict(softcap=2.0), dict(slopes=True), dict(softcap=5.0, slopes=True, causal=False), dict(prefix=[0, 70]), dict(prefix=[190, -4]),
    dict(prefix=[1 << 20, 64], softcap=1.0), dict(documents=1), dict(documents=2, causal=False), dict(documents=3, prefix=[100, 130], slopes=True),
    dict(documents=4, softcap=3.0, slopes=True), dict(scale=0.0), dict(scale=-0.7, slopes=True),
], ids=lambda kw: "-".join(kw))
def test_masks(kw, D):
    B, S, H = 2, 190, 4
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = SLOPES(H)
    if "prefix" in kw:
        kw["prefix"] = torch.tensor(kw["prefix"], dtype=torch.int32)
    if "documents" in kw:
        kw["documents"] = documents(B, S, kw["documents"])
    compare(case(B, S, H, 2, D, BF, 77), BF, **kw)


def test_more_tiles_than_one_look():
    """Past 64 tiles of 64 keys: causal, a prefix, and documents whose tiles lie far apart."""
    S = 4500
    t = case(1, S, 2, 1, 32, BF, 5)
    docs = torch.zeros(1, S, dtype=torch.int32)
    docs[0, 100:4300] = torch.arange(4200, dtype=torch.int32) // 300 + 1
    docs[0, 4400:] = -1
    compare(t, BF, documents=docs)
    compare(t, BF, prefix=torch.tensor([4200], dtype=torch.int32))


@pytest.mark.parametrize("D", [24, 72, 128])
def test_long_sequences(D):
    """Ten looks of 64 tiles and more, two heads that share keys, a prefix and documents, against sums in float64 that never
    hold more than some rows of scores.  An operand of a product (P, dz) is off by half a step of bf16, 2^-8 of it (8 bits:
    steps of 2^-7 of the power of two below), as is a result.  delta = do o takes o as the rounded P made it: it is off by
    that of |do| P |v|, and dz by P times as much.  P = 2^(z - L) by the rounding of z and L in fp32, |z| and |L| below 64
    here: 2^-24 * 128 ln 2 < 2^-17, and with it dz before it cancels, dP and delta being sums of D <= 128 products in fp32
    (2^-17 of their absolute sums, as o's two halves)."""
    S, H, step, half, tail = 41_000, 2, 500, torch.finfo(BF).eps / 2, 2.0 ** -16
    t = case(1, S, H, 1, D, BF, D)
    docs = (torch.arange(S, dtype=torch.int32) // 17_000)[None].clone()
    docs[0, 30_000:30_100] = 0
    docs[0, -70:] = -1
    prefix = 2_500
    got = {n: v[0].double() for n, v in run(t, documents=docs, prefix=torch.tensor([prefix], dtype=torch.int32)).items()}
    q, k, v, dy = (t[n][0].cuda().double() for n in ("q", "k", "v", "dy"))
    k, v, docs, at = k[:, 0], v[:, 0], docs[0].cuda(), torch.arange(S, device="cuda")
    scale = D ** -0.5
    dk, dv, dk_off, dv_off = (torch.zeros(S, D, dtype=torch.float64, device="cuda") for _ in range(4))

    def near(a, b, off):
        assert bool(((a - b).abs() <= off + half * (b.abs() + off) + 2.0 ** -120).all())

    for i in range(0, S, step):
        r = slice(i, i + step)
        seen = ((at[r, None] >= at) | (at < prefix)) & (docs[r, None] == docs) & (docs[r, None] >= 0)
        for h in range(H):
            z = (q[r, h] @ k.t() * scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(z, -1).nan_to_num(0.0)
            o, g = p @ v, dy[r, h]
            near(got["y"][r, h], o, (half + tail) * (p @ v.abs()))
            dp, delta = g @ v.t(), (g * o).sum(-1, keepdim=True)
            dz = p * (dp - delta)
            of_delta = (g.abs() * (p @ v.abs())).sum(-1, keepdim=True)
            off = half * dz.abs() + p * (tail * (g.abs() @ v.abs().t()) + (half + tail) * of_delta)
            near(got["q"][r, h], scale * dz @ k, scale * off @ k.abs())
            dk += scale * dz.t() @ q[r, h]
            dk_off += scale * off.t() @ q[r, h].abs()
            dv += p.t() @ g
            dv_off += (half + tail) * (p.t() @ g.abs())
    near(got["k"][:, 0], dk, dk_off)
    near(got["v"][:, 0], dv, dv_off)


def test_packed_documents_are_their_own_sequences():
    """Each document's rows are, to the bit, not those of another batch, but within the bounds of its own sequence."""
    t = case(1, 330, 2, 2, 64, BF, 9)
    lengths = [1, 64, 129, 100, 36]
    docs = torch.repeat_interleave(torch.arange(5), torch.tensor(lengths))[None]
    got = run(t, documents=docs)
    at = 0
    for n in lengths:
        part = {m: v[:, at:at + n] for m, v in t.items()}
        check({m: v[:, at:at + n] for m, v in got.items()}, want(part, BF))
        at += n


@pytest.mark.parametrize("kw", [dict(), dict(causal=False, softcap=4.0)])
def test_padding_may_hold_anything(kw):
    """NaN and infinities in rows without a document, in q, k, v and the gradient from above, reach nothing; zeros come out."""
    B, S = 2, 200
    t = case(B, S, 4, 2, 128, HF, 12)
    docs = torch.zeros(B, S, dtype=torch.int64)
    docs[0, 150:] = -1
    docs[1, :20] = -7
    docs[1, 90:] = 3
    plain = compare(t, HF, documents=docs, **kw)
    for bad in (math.nan, math.inf):
        for n in t:
            t[n][docs < 0] = bad
        got = run(t, documents=docs, **kw)
        assert all(torch.equal(got[n], plain[n]) for n in got)
        assert not any(got[n].cpu()[docs < 0].any() for n in got)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [1, 40, 64, 96, 128])
def test_one_key_has_no_gradient_of_its_score(D, dtype):
    """A probability of 1 whatever the score: o is v and dq and dk are zeros, not what is left of a difference."""
    for B, S, kw in ((3, 1, dict()), (1, 1, dict(softcap=50.0, prefix=torch.tensor([1], dtype=torch.int32))),
                     (2, 77, dict(documents=torch.arange(77)[None].expand(2, 77), causal=False))):
        t = case(B, S, 8, 2, D, dtype, D + S)
        got = run(t, **kw)
        assert torch.equal(got["y"].cpu(), t["v"].repeat_interleave(4, 2)) and not got["q"].any() and not got["k"].any()
        check({"v": got["v"]}, {"v": want(t, dtype, **kw)["v"]})


@pytest.mark.parametrize("D", [64, 80, 128])
def test_a_prefix_says_nothing_without_the_causal_mask(D):
    t = case(2, 150, 4, 2, D, BF, D)
    docs = documents(2, 150, D)
    for kw in (dict(), dict(documents=docs), dict(slopes=SLOPES(4), softcap=2.0)):
        plain = run(t, causal=False, **kw)
        got = run(t, causal=False, prefix=torch.tensor([70, -3]), **kw)
        assert all(torch.equal(got[n], plain[n]) for n in plain)


@pytest.mark.parametrize("scale,cap", [(0.0, 0.0), (1e-6, 0.0), (-30.0, 0.0), (0.0, 3.0)])
def test_slopes_beside_small_and_large_scales(scale, cap):
    """Slopes of either sign, none, and one so steep that a query sees itself alone."""
    t = case(2, 140, 4, 2, 64, BF, 31, scale=0.4)
    compare(t, BF, scale=scale, softcap=cap, slopes=torch.tensor([0.5, 0.0, -0.03, 1e6]))


def test_nothing_but_padding():
    t = case(1, 130, 2, 1, 64, BF, 13)
    got = run(t, documents=torch.full((1, 130), -1))
    assert not any(v.any() for v in got.values())


def test_large_scores():
    """Rows whose softmax is one key's, scores of hundreds (the running maximum moves many times), and of -hundreds."""
    t = case(1, 260, 2, 1, 64, BF, 14)
    t["k"] = t["k"] * torch.linspace(0, 3, 260).to(BF)[None, :, None, None]
    for scale in (4.0, -4.0):
        got = compare(t, BF, scale=scale)
        assert all(torch.isfinite(v).all() for v in got.values())


def test_a_nan_stays_in_rows_that_see_it():
    t = case(1, 300, 1, 1, 64, BF, 15)
    t["v"][0, 200, 0, 3] = math.nan
    y = run(t)["y"].cpu()
    assert torch.isfinite(y[0, :192]).all() and torch.isnan(y[0, 200:, 0, 3]).all()  # (tiles of 64)


def test_strides():
    """Slices of one projection, heads in front, an expanded key head, rows that start unaligned; gradients too."""
    B, S, H, KV, D = 2, 100, 4, 2, 64
    t = case(B, S, H, KV, D, BF, 16)
    plain = run(t)
    packed = torch.cat([t["q"], t["k"], t["v"]], 2).cuda()
    forms = {
        "packed": dict(zip("qkv", packed.split([H, KV, KV], 2))),
        "heads first": {n: t[n].cuda().transpose(1, 2).contiguous().transpose(1, 2) for n in "qkv"},
        "unaligned": {n: torch.zeros(t[n].numel() + 3, dtype=BF, device="cuda")[3:].view(t[n].shape).copy_(t[n]) for n in "qkv"},
        "pitch": {n: torch.zeros(*t[n].shape[:3], D + 4, dtype=BF, device="cuda")[..., :D].copy_(t[n]) for n in "qkv"},
        "reversed": {n: t[n].cuda().transpose(2, 3).contiguous().transpose(2, 3) for n in "qkv"},
    }
    for name, form in forms.items():
        leaves = {n: v.detach().requires_grad_(True) for n, v in form.items()}
        y = orda.masked_attention(**leaves)
        dy = t["dy"].cuda().transpose(1, 2).contiguous().transpose(1, 2)
        got = {"y": y, **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))}
        assert all(torch.equal(got[n], plain[n]) for n in plain), name
    one = t["k"][:, :, :1].cuda()
    y = orda.masked_attention(t["q"].cuda(), one.expand(B, S, H, D), one.expand(B, S, H, D))
    assert torch.equal(y, orda.masked_attention(t["q"].cuda(), one, one))
    dy = torch.ones((), dtype=BF, device="cuda").expand(B, S, H, D)  # (what sum() hands back)
    leaves = [t[n].cuda().requires_grad_(True) for n in "qkv"]
    y = orda.masked_attention(*leaves)
    a = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    b = torch.autograd.grad(y, leaves, dy.contiguous())
    assert all(torch.equal(x, z) for x, z in zip(a, b))


def test_gradients_one_at_a_time():
    t = case(2, 140, 4, 2, 72, BF, 17)
    docs = documents(2, 140, 5).cuda()
    leaves = {n: t[n].cuda().requires_grad_(True) for n in "qkv"}
    every = torch.autograd.grad(orda.masked_attention(**leaves, documents=docs), list(leaves.values()), t["dy"].cuda())
    for name, full in zip("qkv", every):
        some = {n: t[n].cuda().requires_grad_(n == name) for n in "qkv"}
        (g,) = torch.autograd.grad(orda.masked_attention(**some, documents=docs), some[name], t["dy"].cuda())
        assert torch.equal(g, full)


def test_the_same_tensor_as_query_key_and_value():
    x = torch.randn(1, 90, 2, 64, device="cuda").to(BF)
    leaves = [x.clone().requires_grad_(True) for _ in range(3)]
    one = x.clone().requires_grad_(True)
    dy = torch.randn_like(x)
    parts = torch.autograd.grad(orda.masked_attention(*leaves), leaves, dy)
    (g,) = torch.autograd.grad(orda.masked_attention(one, one, one), one, dy)
    assert torch.allclose(g.float(), sum(p.float() for p in parts), atol=2.0 ** -6 * float(g.abs().max()))


def test_results_do_not_depend_on_the_run():
    t = case(2, 700, 8, 2, 128, BF, 18)
    first = run(t, softcap=20.0)
    for _ in range(3):
        assert all(torch.equal(first[n], v) for n, v in run(t, softcap=20.0).items())


def test_long_strides_and_offsets():
    """Heads of tensors of more than 2^32 bytes, and positions up to 2^22 elements apart; further apart, they are copied."""
    t = case(1, 130, 2, 1, 64, BF, 19)
    plain = run(t)
    for pitch in (1 << 22, (1 << 22) + 64):
        far = torch.zeros(130 * pitch + 64 * 4, dtype=BF, device="cuda")
        assert far.numel() * 2 > 1 << 30
        at = far.as_strided((1, 130, 4, 64), (0, pitch, 64, 1))
        at.copy_(torch.cat([t["q"], t["k"], t["v"]], 2))
        leaves = {n: v.detach().requires_grad_(True) for n, v in zip("qkv", at.split([2, 1, 1], 2))}
        y = orda.masked_attention(**leaves)
        got = {"y": y, **dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())))}
        assert all(torch.equal(got[n], plain[n]) for n in plain)
    big = torch.zeros(40, 130, 4, 1 << 17, dtype=BF, device="cuda")  # (batches 2^26 elements apart: 40 of them pass 2^32 bytes)
    b = big[..., 64:128]
    b[39] = torch.cat([t["q"], t["k"], t["v"]], 2)[0].cuda()
    y = orda.masked_attention(b[:, :, :2], b[:, :, 2:3], b[:, :, 3:])
    assert torch.equal(y[39], plain["y"][0])


@pytest.mark.parametrize("call,match", [
    (lambda q: orda.masked_attention(q.float(), q.float(), q.float()), "bfloat16 and float16"),
    (lambda q: orda.masked_attention(*[torch.zeros(1, 3, 1, 136, device="cuda", dtype=BF)] * 3), "head_dim up to 128"),
    (lambda q: orda.masked_attention(q, q, q, documents=torch.zeros(1, 3, dtype=torch.int32)), "documents is on cpu"),
])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call(torch.zeros(1, 3, 1, 8, device="cuda", dtype=BF))


def test_fp32_under_autocast_and_in_torch():
    t = case(1, 40, 2, 1, 64, BF, 20)
    leaves = {n: t[n].cuda().float().requires_grad_(True) for n in "qkv"}
    with torch.autocast("cuda", dtype=BF):
        y = orda.masked_attention(**leaves)
    grads = torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())
    assert y.dtype == BF and all(g.dtype == torch.float32 for g in grads)
    check({"y": y, **dict(zip(leaves, grads))}, want(t, BF))
    z = orda.masked_attention(**leaves, backend="torch")
    assert z.dtype == torch.float32 and float((z - y.float()).abs().max()) < 0.05
