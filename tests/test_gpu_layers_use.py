"""The projection, the feed-forward block and clipping as programs call them: mixed dtypes, autocast, checkpointing, shared
tensors, streams, captured graphs, second derivatives, very long and very wide tensors."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

import orda_ce_kernel as orda
from tests._layers import Unit, check, random_inputs
from tests.test_gpu_layers import ffn_case, linear_case, run_ffn, run_linear, want_ffn, want_linear

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("N", [4, 90])
def test_mixed_dtypes(N):
    """fp32 master weights beside bf16 activations: computed in bf16 on the rounded weights, every gradient in its own
    tensor's dtype (the bf16 gradient's value)."""
    t = linear_case(N, 96, 77, BF, "silu", True, True, seed=20)
    wide = {**t, "w": t["w"].float() * (1 + 2.0 ** -12), "bias": t["bias"].float()}
    assert torch.equal(wide["w"].to(BF), t["w"])  # (an eighth of half a step off)
    got = run_linear(wide, "silu")
    assert got["y"].dtype == got["x"].dtype == BF and got["w"].dtype == got["bias"].dtype == torch.float32
    check(got, want_linear(t, "silu", BF))
    f = ffn_case(N, 96, 72, 88, BF, "silu", True, seed=21)
    got = run_ffn({**f, "w_up": f["w_up"].float(), "w_down": f["w_down"].float()}, "silu")
    assert got["w_up"].dtype == torch.float32 and got["w_gate"].dtype == BF
    check(got, want_ffn(f, "silu", BF))


def test_autocast():
    t = linear_case(90, 96, 77, torch.float16, "gelu", True, False, seed=22)
    leaves = {n: v.cuda().float().requires_grad_(True) for n, v in t.items() if n != "dy"}
    with torch.autocast("cuda", dtype=torch.float16):
        y = orda.fused_linear(leaves["x"], leaves["w"], leaves["bias"], activation="gelu")
    grads = torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())
    assert y.dtype == torch.float16 and all(g.dtype == torch.float32 for g in grads)
    check({"y": y, **dict(zip(leaves, grads))}, want_linear(t, "gelu", torch.float16))


def test_differentiable_once():
    t = ffn_case(20, 96, 72, 88, BF, "silu", False, seed=23)
    x, wg, wu, wd = (t[n].cuda().requires_grad_(True) for n in ("x", "w_gate", "w_up", "w_down"))
    for y in (orda.gated_feed_forward(x, wg, wu, wd), orda.fused_linear(x, wg, activation="silu")):
        (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()


def test_forward_mode_and_transforms_are_refused():
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="jvp"):
            orda.fused_linear(forward_ad.make_dual(x, torch.ones_like(x)), w)
        with pytest.raises(RuntimeError, match="jvp"):
            orda.gated_feed_forward(forward_ad.make_dual(x, torch.ones_like(x)), w, w, w.t().contiguous())
    for transform in (torch.func.grad, torch.func.vmap):
        with pytest.raises(RuntimeError):
            transform(lambda a: orda.fused_linear(a, w, activation="silu").sum())(x)


def test_checkpointing_and_changed_operands():
    t = ffn_case(40, 96, 72, 88, BF, "silu", True, seed=24)
    plain = run_ffn(t, "silu")
    leaves = {n: v.cuda().requires_grad_(True) for n, v in t.items() if n != "dy"}
    y = checkpoint(orda.gated_feed_forward, *[leaves[n] for n in ("x", "w_gate", "w_up", "w_down", "residual")], use_reentrant=False)
    y.backward(t["dy"].cuda())
    assert torch.equal(y, plain["y"]) and all(torch.equal(v.grad, plain[n]) for n, v in leaves.items())
    w = leaves["w_gate"].detach().clone().requires_grad_(True)
    y = orda.fused_linear(leaves["x"].detach(), w, activation="silu")
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_inside_compiled_code_and_inference_mode():
    """A compiled caller breaks its graph at the call and gives the same bits; inference mode records nothing."""
    t = linear_case(40, 96, 72, BF, "gelu", True, False, seed=33)
    x, w, b = (t[n].cuda().requires_grad_(True) for n in ("x", "w", "bias"))

    def f(x, w, b):
        return orda.fused_linear(x * 2, w, b, activation="gelu") + 1

    y, z = f(x, w, b), torch.compile(f, backend="eager")(x, w, b)
    assert torch.equal(y, z)
    for one, two in zip(torch.autograd.grad(y, (x, w, b), t["dy"].cuda()), torch.autograd.grad(z, (x, w, b), t["dy"].cuda())):
        assert torch.equal(one, two)
    with torch.inference_mode():
        v = f(x, w, b)
    assert torch.equal(v, y) and v.grad_fn is None and v.is_inference()


def test_the_same_tensor_in_two_places():
    """One weight as gate and up, x as the residual, a square weight as its own input: gradients add up."""
    t = ffn_case(90, 96, 72, 96, BF, "silu", True, seed=25)
    t["w_up"], t["residual"] = t["w_gate"], t["x"]
    want = want_ffn(t, "silu", BF)
    x, w, wd = (t[n].cuda().requires_grad_(True) for n in ("x", "w_gate", "w_down"))
    y = orda.gated_feed_forward(x, w, w, wd, x)
    y.backward(t["dy"].cuda())
    q = Unit(BF)

    def both(a, b):  # (each rounded, then their sum)
        v = want[a][0] + want[b][0]
        return v, want[a][1] + want[b][1] + q.rounded(v) * 1.01

    check({"y": y, "x": x.grad, "w": w.grad, "w_down": wd.grad},
          {"y": want["y"], "x": both("x", "residual"), "w": both("w_gate", "w_up"), "w_down": want["w_down"]})
    s = random_inputs({"x": ((72, 72), 0.2), "dy": ((72, 72), 1.0)}, BF, 26)
    s["w"] = s["x"]
    want = want_linear(s, "none", BF)
    a = s["x"].cuda().requires_grad_(True)
    y = orda.fused_linear(a, a)
    y.backward(s["dy"].cuda())
    check({"y": y, "x": a.grad}, {"y": want["y"], "x": both("x", "w")})


def test_two_streams_at_once():
    """Calls in flight on two streams give what each gives alone."""
    cases = [ffn_case(300, 264, 520, 264, BF, "silu", True, seed=s) for s in (27, 28)]
    alone = [run_ffn(c, "silu") for c in cases]
    grads = [[torch.randn(1000, 77, device="cuda") for _ in range(9)] for _ in range(2)]
    norms = [orda.grad_norm(g).clone() for g in grads]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got, total = [], []
        for c, g, s in zip(cases, grads, streams):
            with torch.cuda.stream(s):
                got.append(run_ffn(c, "silu"))
                total.append(orda.grad_norm(g))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(a[n], b[n]) for n in a)
        assert all(torch.equal(a, b) for a, b in zip(norms, total))


def test_captured_backward_beside_an_eager_graph_of_the_same_leaves():
    """On the default stream's graph the captured backward pass is refused with an error; once that graph is gone, or with
    leaves of its own, it runs."""
    w = torch.randn(24, 16, device="cuda", requires_grad=True)
    x = torch.randn(40, 16, device="cuda")
    eager = orda.fused_linear(x, w, activation="silu").sum()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (warm)
        own = w.detach().requires_grad_(True)
        torch.autograd.grad(orda.fused_linear(x, own, activation="silu").sum(), own)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = orda.fused_linear(x, w, activation="silu").sum()
        with pytest.raises(RuntimeError, match="same leaf"):
            torch.autograd.grad(y, w)
        own = w.detach().requires_grad_(True)
        (got,) = torch.autograd.grad(orda.fused_linear(x, own, activation="silu").sum(), own)
    graph.replay()
    torch.cuda.synchronize()
    (want,) = torch.autograd.grad(eager, w)
    assert torch.equal(got, want)


@pytest.mark.parametrize("N", [3, 40])
def test_rows_very_far_apart(N):
    """A pitch past what the C entry points take: the rows are copied."""
    t = linear_case(N, 96, 77, BF, "none", False, True, seed=29)
    far = torch.zeros(N, (1 << 22) + 64, dtype=BF, device="cuda")
    far[:, :96] = t["x"].cuda()
    far[:, 100:177] = t["residual"].cuda()
    leaves = [v.requires_grad_(True) for v in (far[:, :96].detach(), t["w"].cuda(), far[:, 100:177].detach())]
    y = orda.fused_linear(leaves[0], leaves[1], None, leaves[2])
    got = torch.autograd.grad(y, leaves, t["dy"].cuda())
    check({"y": y, "x": got[0], "w": got[1], "residual": got[2]}, want_linear(t, "none", BF))


@pytest.mark.parametrize("K,O", [(1 << 21, 24), (24, 1 << 21)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_widest_layers(K, O, dtype):
    """Rows of 2^21 elements, two tiles of them: 256 rows of an fp32 output span 2^32 bytes.  Small whole numbers, exact
    sums."""
    N = 300
    g = torch.Generator(device="cuda").manual_seed(31)

    def whole(*shape):
        return torch.randint(-1, 2, shape, generator=g, device="cuda", dtype=torch.int8).to(dtype)

    x, w, r, dy = whole(N, K).requires_grad_(True), whole(O, K).requires_grad_(True), whole(N, O), whole(N, O)
    y = orda.fused_linear(x, w, None, r, activation="relu")
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    q = Unit(dtype)
    with torch.no_grad():
        for a in range(0, O, 1 << 18):
            b = slice(a, min(O, a + (1 << 18)))
            z = x.float() @ w[b].float().t()  # (whole numbers below 2^24: exact in fp32)
            want = z.clamp(min=0) + r[:, b].float()
            assert bool(((y[:, b].float() - want).abs() <= q.rounded(want)).all())
            dz = dy[:, b].float() * (z > 0)
            dw = dz.t() @ x.float()
            assert bool(((gw[b].float() - dw).abs() <= q.rounded(dw)).all())
            part = dz @ w[b].float()
            total = part if a == 0 else total + part
        assert bool(((gx.float() - total).abs() <= q.rounded(total)).all())


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_offsets_past_32_bits(dtype):
    """x and its gradient of more than 2^32 bytes (16-bit: K of the weight's gradient in ranges of at most 2^30 bytes).
    Small whole numbers: every product and sum is exact below 2^24, so what is left is each output's rounding."""
    K, O = 2056, 40
    N = ((1 << 32) + (1 << 28)) // (K * dtype.itemsize) + 5
    g = torch.Generator(device="cuda").manual_seed(30)

    def whole(*shape):
        return torch.randint(-2, 3, shape, generator=g, device="cuda", dtype=torch.int8).to(dtype)

    x, w, dy = whole(N, K).requires_grad_(True), whole(O, K).requires_grad_(True), whole(N, O)
    y = orda.fused_linear(x, w, activation="relu")
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    q, total = Unit(dtype), torch.zeros(O, K, dtype=torch.float64, device="cuda")

    def same(got, want):
        assert bool(((got.double() - want).abs() <= q.rounded(want)).all())

    for a in range(0, N, 1 << 17):
        b = slice(a, min(N, a + (1 << 17)))
        xb = x[b].detach().double()
        z = xb @ w.detach().double().t()
        dz = dy[b].double() * (z > 0)
        same(y[b].detach(), z.clamp(min=0))
        same(gx[b], dz @ w.detach().double())
        total += dz.t() @ xb
    assert float(total.abs().max()) < 2 ** 24
    same(gw, total)


def test_block_offsets_past_32_bits():
    """h, the kept factors, da and db of more than 2^31 elements each.  Values -1, 0, 1: a, b, h and the factors are whole
    numbers below 2^8, every sum stays below 2^24, so only outputs round."""
    H, F, O = 8, 2048, 8
    N = (1 << 31) // F + 70
    g = torch.Generator(device="cuda").manual_seed(32)

    def whole(*shape):
        return torch.randint(-1, 2, shape, generator=g, device="cuda", dtype=torch.int8).to(BF)

    t = [whole(N, H), whole(F, H), whole(F, H), whole(O, F)]
    leaves = [v.requires_grad_(True) for v in t]
    dy = whole(N, O)
    y = orda.gated_feed_forward(*leaves, activation="relu")
    grads = torch.autograd.grad(y, leaves, dy)
    q = Unit(BF)

    def same(got, want):
        assert bool(((got.float() - want).abs() <= q.rounded(want)).all())

    with torch.no_grad():
        x, wg, wu, wd = (v.detach().float() for v in leaves)
        sums = [torch.zeros_like(w) for w in (wg, wu, wd)]
        for k in range(0, N, 1 << 16):
            b = slice(k, min(N, k + (1 << 16)))
            a, u, d = x[b] @ wg.t(), x[b] @ wu.t(), dy[b].float() @ wd
            f = a.clamp(min=0)
            same(y[b], (f * u) @ wd.t())
            da, db = d * u * (a > 0), d * f
            same(grads[0][b], da @ wg + db @ wu)
            for s, v in zip(sums, (da.t() @ x[b], db.t() @ x[b], dy[b].float().t() @ (f * u))):
                s += v
        for got, want in zip(grads[1:], sums):
            assert float(want.abs().max()) < 2 ** 24
            same(got, want)
