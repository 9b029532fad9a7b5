"""Measured cases of the operators that a student's training step needs around its projections: the token embedding, dropout,
the layer norm with dropout and residual in front of it, and masked self-attention.

A case names the operator (``op``), its sizes and options; ``prepare`` makes what the program holds before the call, ``run``
is one pass (forward, and for a training case its backward).  With ``own`` false the pass is written in elementary torch
operations in fp32, rounded once at the end; with ``own`` true it calls this package.  Sizes are the framework's own
configurations (hidden 256 to 5120, vocabularies 32000 to 152064, 512 to 16384 tokens) and generic ones between and beside
them.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

GRAD_SCALE = 0.1  # of the gradients that come from above
EPS = 1e-5


def _orda():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "orda-knowledge-distillation-kernel_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import orda_ce_kernel

    return orda_ce_kernel


# ------------------------------------------------------------------- cases
def _embed(N, V, H, **kw):
    return dict(dict(op="embed", N=N, V=V, H=H, dtype="bfloat16", scaled=False, pad=0.0, train=False), **kw)


def _drop(N, H, **kw):
    return dict(dict(op="dropout", N=N, H=H, dtype="bfloat16", p=0.1, residual=False, train=False), **kw)


def _norm(N, H, **kw):
    return dict(dict(op="norm", N=N, H=H, dtype="bfloat16", params="same", bias=True, residual=False, p=0.0, train=False), **kw)


def _attn(B, S, H, KV, D, **kw):
    return dict(dict(op="attention", B=B, S=S, H=H, KV=KV, D=D, dtype="bfloat16", causal=True, softcap=0.0, slopes=False,
                     documents=0, prefix=False, train=False), **kw)


def listed():
    return [
        # a micro-batch of a student in evaluation
        dict(_embed(512, 32000, 1024), name="embed_microbatch"),
        # padded sequences of odd sizes, fp16, the embedding scaled by the root of its width
        dict(_embed(1999, 50257, 777, dtype="float16", scaled=True, pad=0.15, train=True), name="embed_ragged_fp16"),
        # a full batch over a large vocabulary
        dict(_embed(16384, 128256, 4096, train=True), name="embed_train"),
        # a projection's output of a small student, fp32, odd width
        dict(_drop(777, 1001, dtype="float32", p=0.25, train=True), name="dropout_ragged_fp32"),
        # a large batch's output added to the residual stream
        dict(_drop(16384, 4096, residual=True, train=True), name="dropout_add_train"),
        # a micro-batch in evaluation: one norm between two small layers
        dict(_norm(512, 1024), name="norm_microbatch"),
        # padding-free sequences of odd sizes, dropout and residual in front, fp32 parameters beside fp16 activations
        dict(_norm(1999, 1111, dtype="float16", params="float32", residual=True, p=0.1, train=True), name="norm_ragged_fp16"),
        # a full batch of a large student
        dict(_norm(16384, 4096, residual=True, p=0.1, train=True), name="norm_train"),
        # a short sequence in evaluation, no causal mask
        dict(_attn(2, 128, 8, 8, 64, causal=False), name="attention_short"),
        # documents packed into rows with padding behind them, scores capped, odd sizes, fp16
        dict(_attn(3, 1777, 12, 4, 80, dtype="float16", softcap=30.0, documents=7, train=True), name="attention_packed_fp16"),
        # prompts that see themselves whole, scores biased by distance
        dict(_attn(2, 2048, 16, 16, 64, slopes=True, prefix=True, train=True), name="attention_prefix"),
        # a large student's causal attention with shared heads: the largest call
        dict(_attn(2, 4096, 32, 8, 128, train=True), name="attention_train"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A layer's width: mostly multiples of 64, some of 8, a few odd."""
    n, step = _log_int(rng, lo, hi), rng.choice([64, 64, 64, 64, 64, 64, 8, 8, 2, 1])
    return min(hi, max(lo, (n + step - 1) // step * step))


def draw(rng):
    op = rng.choice(["embed", "embed", "dropout", "norm", "norm", "norm", "attention", "attention", "attention"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    train = rng.random() < 0.7
    if op == "attention":
        dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
        B, S = rng.choice([1, 1, 2, 3, 4]), _log_int(rng, 1, 4096)
        KV, group = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 1, 2, 3, 4, 8])
        group = max(1, min(group, 64 // (B * KV)))
        documents = rng.choice([0, 0, 1, _log_int(rng, 1, 16)])
        return _attn(B, S, KV * group, KV, rng.choice([128, 128, 64, 64, 64, 32, 96, 80, 8 * rng.randint(1, 16), rng.randint(1, 128)]),
                     dtype=dtype, causal=rng.random() < 0.8, softcap=rng.choice([0.0, 0.0, 15.0, 50.0]), slopes=rng.random() < 0.3,
                     documents=min(documents, S), prefix=rng.random() < 0.3, train=train)
    N = _log_int(rng, 1, 16384)
    if op == "embed":
        V = _log_int(rng, 500, 152064)
        return _embed(N, V, _width(rng, 64, min(5120, 128256 * 4096 // V)), dtype=dtype, scaled=rng.random() < 0.4,
                      pad=rng.choice([0.0, 0.0, 0.05, 0.4]), train=train)
    H = _width(rng, 8, 5120 if dtype != "float32" else 4096)
    if op == "dropout":
        return _drop(min(N, 16384 * 4096 // H), H, dtype=dtype, p=rng.choice([0.1, 0.1, 0.5, rng.random()]),
                     residual=rng.random() < 0.6, train=train)
    residual = rng.random() < 0.6
    return _norm(min(N, 16384 * 4096 // H), H, dtype=dtype, params=rng.choice(["same", "same", "float32"]), bias=rng.random() < 0.8,
                 residual=residual, p=rng.choice([0.0, 0.1, 0.3]) if residual else 0.0, train=train)


# ------------------------------------------------------------------- inputs
def _spans(case):
    """The documents of each row of an attention case, [(first, end), ...], and its prefix length: of random lengths, with
    padding behind the last.  By the case alone, so that its work is known."""
    rng = random.Random(case["S"] * 1_000_003 + case["B"] * 101 + case["documents"])
    rows = []
    for _ in range(case["B"]):
        S, n = case["S"], case["documents"]
        spans = [(0, S)]
        if n:
            end = max(n, S - int(S * rng.uniform(0.0, 0.1)))
            cuts = [0, *sorted(rng.sample(range(1, end), n - 1)), end]
            spans = list(zip(cuts[:-1], cuts[1:]))
        rows.append((spans, rng.randint(0, S) if case["prefix"] else 0))
    return rows


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = getattr(torch, case["dtype"])

    def rand(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)

    if case["op"] == "embed":
        N, V, H = case["N"], case["V"], case["H"]
        # word frequencies that fall with the rank, the ranks spread over the vocabulary; padding at the end
        rank = torch.rand(N, generator=g, device="cuda", dtype=torch.float64).mul(math.log(V)).exp().long().clamp(1, V) - 1
        ids = (rank * 7919 + 17) % V
        if case["pad"]:
            ids[N - int(case["pad"] * N):] = 0
        t = {"ids": ids, "w": rand(V, H, scale=H ** -0.5 if case["scaled"] else 1.0)}
        if case["train"]:
            t["dy"] = rand(N, H, scale=GRAD_SCALE)
        return t
    if case["op"] == "dropout":
        t = {"x": rand(case["N"], case["H"])}
        if case["residual"]:
            t["residual"] = rand(case["N"], case["H"])
        if case["train"]:
            t["dy"] = rand(case["N"], case["H"], scale=GRAD_SCALE)
        return t
    if case["op"] == "norm":
        N, H = case["N"], case["H"]
        pt = torch.float32 if case["params"] == "float32" else dt
        # a residual stream: a few channels far from zero, and an offset
        t = {"x": rand(N, H), "w": rand(H, scale=0.1, dtype=pt).add_(1.0)}
        if case["bias"]:
            t["bias"] = rand(H, scale=0.1, dtype=pt)
        channels = torch.where(torch.rand(H, generator=g, device="cuda") < 0.02, 8.0, 1.0).to(dt)
        if case["residual"]:
            t["residual"] = rand(N, H).mul_(channels).add_(0.25)
        else:
            t["x"] = t["x"].mul_(channels).add_(0.25)
        if case["train"]:
            t["dy"] = rand(N, H, scale=GRAD_SCALE)
            if case["residual"]:
                t["ds"] = rand(N, H, scale=GRAD_SCALE)
        return t
    B, S, H, KV, D = (case[n] for n in ("B", "S", "H", "KV", "D"))
    # one projection's output: queries, keys and values side by side
    qkv = rand(B, S, H + 2 * KV, D)
    q, k, v = qkv.split([H, KV, KV], dim=2)
    t = {"q": q, "k": k, "v": v}
    if case["slopes"]:
        t["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)
    rows = _spans(case)
    if case["documents"]:
        ids = torch.full((B, S), -1, dtype=torch.int32)
        for b, (spans, _) in enumerate(rows):
            for i, (first, end) in enumerate(spans):
                ids[b, first:end] = i
        t["documents"] = ids.cuda()
    if case["prefix"]:
        t["prefix"] = torch.tensor([p for _, p in rows], dtype=torch.int32, device="cuda")
    if case["train"]:
        t["dy"] = rand(B, S, H, D, scale=GRAD_SCALE)
    return t


_LEAVES = {"embed": ("w",), "dropout": ("x", "residual"), "norm": ("x", "residual", "w", "bias"), "attention": ("q", "k", "v")}


def _seed_of(seed):
    """The seed of a case's dropout, 64 bits."""
    return random.Random(int(seed)).getrandbits(63)


def prepare(case, seed):
    t = _inputs(case, seed)
    leaves = [n for n in _LEAVES[case["op"]] if n in t]
    if case["train"]:
        for n in leaves:
            t[n] = t[n].detach().requires_grad_(True)
    return {"case": case, "t": t, "leaves": leaves, "seed": _seed_of(seed)}


# ------------------------------------------------------------------- plain form
def _kept(n, p, seed, device):
    """1 / (1 - p) for the elements that are kept, 0 for the others: 16 bits of Philox4x32-10 (key: the seed, counter: the
    element's index / 8 and the site, here 0) against p in steps of 2^-16.  Whole numbers of 64 bits hold the products."""
    mask = 0xFFFFFFFF
    drop = math.floor(p * 65536 + 0.5)
    index = torch.arange((n + 7) // 8, device=device)
    c = [index & mask, index >> 32, torch.zeros_like(index), torch.zeros_like(index)]
    k0, k1 = seed & mask, seed >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & mask) ^ c[1] ^ k0, b & mask, ((a >> 32) & mask) ^ c[3] ^ k1, a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack(c, 1)
    u = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]
    return (u >= drop).float() * (65536.0 / (65536 - drop) if drop < 65536 else 0.0)


def _plain_embed(case, t):
    scale = case["H"] ** 0.5 if case["scaled"] else 1.0
    out = {"y": (t["w"][t["ids"]].float() * scale).to(t["w"].dtype)}
    if case["train"]:
        dy = t["dy"].float()
        if case["pad"]:
            dy = dy * (t["ids"] != 0).unsqueeze(1)
        dw = torch.zeros(case["V"], case["H"], device=dy.device).index_add_(0, t["ids"], dy)
        out["w"] = (dw * scale).to(t["w"].dtype)
    return out


def _plain_dropout(case, t, seed):
    dt = t["x"].dtype
    keep = _kept(t["x"].numel(), case["p"], seed, t["x"].device).view_as(t["x"])
    y = t["x"].float() * keep
    if case["residual"]:
        y = y + t["residual"].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        out["x"] = (t["dy"].float() * keep).to(dt)
        if case["residual"]:
            out["residual"] = t["dy"]
    return out


def _plain_norm(case, t, seed):
    dt, pt = t["x"].dtype, t["w"].dtype
    f = {n: v.float() for n, v in t.items()}
    s, keep = f["x"], None
    if case["p"]:
        keep = _kept(s.numel(), case["p"], seed, s.device).view_as(s)
        s = s * keep
    if case["residual"]:
        s = s + f["residual"]
    d = s - s.mean(1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    h = d * rstd
    y = h * f["w"]
    if case["bias"]:
        y = y + f["bias"]
    out = {"y": y.to(dt)}
    if case["residual"]:
        out["s"] = s.to(dt)
    if case["train"]:
        g = f["dy"] * f["w"]
        ds = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        if case["residual"]:
            ds = ds + f["ds"]
        out["x"] = (ds if keep is None else ds * keep).to(dt)
        if case["residual"]:
            out["residual"] = ds.to(dt)
        out["w"] = (f["dy"] * h).sum(0).to(pt)
        if case["bias"]:
            out["bias"] = f["dy"].sum(0).to(pt)
    return out


def _plain_attention(case, t):
    B, S, H, KV, D = (case[n] for n in ("B", "S", "H", "KV", "D"))
    G, dt = H // KV, t["q"].dtype

    def heads(x):  # (B, S, H, D) -> (B KV, G S, D)
        return x.float().view(B, S, KV, -1, D).permute(0, 2, 3, 1, 4).reshape(B * KV, -1, D)

    def back(x):
        return x.view(B, KV, -1, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, -1, D).to(dt)

    q, k, v = heads(t["q"]), heads(t["k"]), heads(t["v"])
    scale = D ** -0.5
    z, th = torch.bmm(q, k.transpose(1, 2).contiguous()) * scale, None
    if case["softcap"]:
        th = torch.tanh(z / case["softcap"])
        z = th * case["softcap"]
    z = z.view(B, KV, G, S, S)
    i = torch.arange(S, device=q.device)
    if case["slopes"]:
        z = z - t["slopes"].view(1, KV, G, 1, 1) * (i[:, None] - i[None]).abs()
    seen = torch.ones(B, 1, 1, S, S, dtype=torch.bool, device=q.device)
    if case["causal"]:
        seen = (i[:, None] >= i[None]).expand_as(seen)
        if case["prefix"]:
            seen = seen | (i < t["prefix"].view(B, 1, 1, 1, 1))
    if case["documents"]:
        doc = t["documents"]
        seen = seen & (doc[:, :, None] == doc[:, None]).view(B, 1, 1, S, S) & (doc >= 0).view(B, 1, 1, S, 1)
    z = z.masked_fill(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    p = (e / total.masked_fill(total == 0.0, 1.0)).view(B * KV, G * S, S)
    o = torch.bmm(p, v)
    out = {"y": back(o)}
    if case["train"]:
        do = heads(t["dy"])
        dp = torch.bmm(do, v.transpose(1, 2).contiguous())
        dz = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
        if th is not None:
            dz = dz * (1.0 - th * th)
        out["q"] = back(torch.bmm(dz, k))
        out["k"] = back(torch.bmm(dz.transpose(1, 2).contiguous(), q))
        out["v"] = back(torch.bmm(p.transpose(1, 2).contiguous(), do))
    return out


# ------------------------------------------------------------------- one pass
def run(state):
    case, t = state["case"], state["t"]
    op = case["op"]
    if not own:
        with torch.no_grad():
            if op == "embed":
                return _plain_embed(case, t)
            if op == "dropout":
                return _plain_dropout(case, t, state["seed"])
            return _plain_norm(case, t, state["seed"]) if op == "norm" else _plain_attention(case, t)
    ys, grads = ("y",), [t["dy"]] if case["train"] else []
    with torch.set_grad_enabled(case["train"]):
        if op == "embed":
            y = _orda().token_embedding(t["ids"], t["w"], scale=case["H"] ** 0.5 if case["scaled"] else 1.0,
                                        padding_idx=0 if case["pad"] else None)
        elif op == "dropout":
            y = _orda().counter_dropout(t["x"], case["p"], t.get("residual"), seed=state["seed"])
        elif op == "norm":
            y = _orda().layer_norm(t["x"], t["w"], t.get("bias"), t.get("residual"), eps=EPS, p=case["p"],
                                   seed=state["seed"] if case["p"] else None)
            if case["residual"]:
                ys, grads = ("y", "s"), grads + ([t["ds"]] if case["train"] else [])
        else:
            y = _orda().masked_attention(t["q"], t["k"], t["v"], causal=case["causal"], softcap=case["softcap"],
                                         slopes=t.get("slopes"), documents=t.get("documents"), prefix=t.get("prefix"))
    y = y if isinstance(y, tuple) else (y,)
    out = {n: v.detach() for n, v in zip(ys, y)}
    if case["train"]:
        out.update(zip(state["leaves"], torch.autograd.grad(y, [t[n] for n in state["leaves"]], grads)))
    return out


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "attention":
        S, D = case["S"], case["D"]
        pairs = 0
        for spans, prefix in _spans(case):
            for first, end in spans:
                n, m = end - first, max(0, min(end, prefix) - first)
                pairs += n * (n + 1) // 2 + m * (m - 1) // 2 if case["causal"] else n * n
        rows = case["B"] * S * (2 * case["H"] + 2 * case["KV"]) * D
        return {"bytes": rows * e * (2 if case["train"] else 1), "flops": 1.0 * pairs * case["H"] * D * (14 if case["train"] else 4)}
    N, H = case["N"], case["H"]
    if case["op"] == "embed":
        n = 2 * N * H * e + 8 * N
        if case["train"]:
            n += (N * H + case["V"] * H) * e
        return {"bytes": n, "flops": (2.0 if case["train"] else 1.0) * N * H}
    r = 1 if case["residual"] else 0
    if case["op"] == "dropout":
        return {"bytes": N * H * e * (2 + r + (2 if case["train"] else 0)), "flops": 8.0 * N * H}
    params = (2 if case["bias"] else 1) * H * (4 if case["params"] == "float32" else e)
    passes = 2 + 2 * r + ((3 + 2 * r) if case["train"] else 0)  # x, y and r, s; s, dy, dx and ds, dr
    if case["train"] and r and not case["p"]:
        passes -= 1  # the residual's gradient is x's
    return {"bytes": N * H * e * passes + params * (3 if case["train"] else 1), "flops": (25.0 if case["train"] else 8.0) * N * H}


# ------------------------------------------------------------------- 64 bits
def _philox(count, key, device):
    """Philox4x32-10's four words for the counters 0 .. count - 1, 32-bit products in halves of 16 bits."""
    def split(x, m):  # (high, low) 32 bits of x m
        ml, mh, xl, xh = m & 0xFFFF, m >> 16, x & 0xFFFF, x >> 16
        low, mid = xl * ml, xh * ml
        mid = mid + (low >> 16)
        second = xl * mh + (mid & 0xFFFF)
        return xh * mh + (mid >> 16) + (second >> 16), ((second & 0xFFFF) << 16) | (low & 0xFFFF)

    n = torch.arange(count, dtype=torch.int64, device=device)
    x = [n % (1 << 32), n // (1 << 32), n * 0, n * 0]
    for r in range(10):
        ka, kb = (key % (1 << 32) + r * 0x9E3779B9) % (1 << 32), (key // (1 << 32) + r * 0xBB67AE85) % (1 << 32)
        (h0, l0), (h1, l1) = split(x[0], 0xD2511F53), split(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ ka, l1, h0 ^ x[3] ^ kb, l0]
    return x


def _factors(shape, p, key, device):
    n = math.prod(shape)
    drop = int(math.floor(65536 * p + 0.5))
    pieces = [piece for w in _philox(-(-n // 8), key, device) for piece in (w % 65536, w // 65536)]
    u = torch.stack(pieces, dim=-1).flatten()[:n].view(shape)
    return torch.where(u < drop, 0.0, 65536.0 / max(65536 - drop, 1)).double()


def exact(case, seed):
    """The definitions in float64, gradients by autograd."""
    t = _inputs(case, seed)
    op, leaves = case["op"], [n for n in _LEAVES[case["op"]] if n in t]
    if op == "attention":
        return _exact_attention(case, t)
    f = {n: v.double() if v.is_floating_point() else v for n, v in t.items()}
    for n in leaves:
        f[n].requires_grad_(case["train"])
    above = [f["dy"]] if case["train"] else []
    if op == "embed":
        y = [torch.nn.functional.embedding(f["ids"], f["w"], padding_idx=0 if case["pad"] else None)
             * (math.sqrt(case["H"]) if case["scaled"] else 1.0)]
    else:
        s = f["x"]
        if case["p"]:
            s = s * _factors(tuple(s.shape), case["p"], _seed_of(seed), s.device)
        if case["residual"]:
            s = f["residual"] + s
        y = [s]
        if op == "norm":
            y = [torch.nn.functional.layer_norm(s, (case["H"],), f["w"], f.get("bias"), EPS)]
            if case["residual"]:
                y, above = y + [s], above + ([f["ds"]] if case["train"] else [])
    out = dict(zip(("y", "s"), (v.detach() for v in y)))
    if case["train"]:
        out.update(zip(leaves, torch.autograd.grad(y, [f[n] for n in leaves], above)))
    return out


def _exact_attention(case, t):
    S, G = case["S"], case["H"] // case["KV"]
    out = {n: torch.empty(t[m].shape, dtype=torch.float64, device="cuda")
           for n, m in (("y", "q"), *((n, n) for n in (("q", "k", "v") if case["train"] else ())))}
    at = torch.arange(S, device="cuda")
    far = (at[:, None] - at[None]).abs().double()
    for b in range(case["B"]):
        hidden = torch.zeros(S, S, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= at[None] > at[:, None]
            if case["prefix"]:
                hidden[:, :int(t["prefix"][b])] = False
        if case["documents"]:
            d = t["documents"][b]
            hidden |= (d[None] != d[:, None]) | (d < 0)[:, None]
        empty = hidden.all(1)
        for h in range(case["H"]):
            q, k, v = (t[n][b, :, i].double().requires_grad_(case["train"]) for n, i in (("q", h), ("k", h // G), ("v", h // G)))
            z = q @ k.t() / math.sqrt(case["D"])
            if case["softcap"]:
                z = case["softcap"] * torch.tanh(z / case["softcap"])
            if case["slopes"]:
                z = z - float(t["slopes"][h]) * far
            z = torch.where(hidden, -math.inf, z)
            p = torch.softmax(torch.where(empty[:, None], 0.0, z), 1)
            o = torch.where(empty[:, None], 0.0, p) @ v
            out["y"][b, :, h] = o.detach()
            if case["train"]:
                for n, g in zip("qkv", torch.autograd.grad(o, (q, k, v), t["dy"][b, :, h].double())):
                    if n == "q":
                        out["q"][b, :, h] = g
                    elif h % G == 0:
                        out[n][b, :, h // G] = g
                    else:
                        out[n][b, :, h // G] += g
    return out
