"""The projection and the gated feed-forward block on the GPU against their definitions in float64, within bounds derived
in tests/_layers.py: every dtype, sizes from one token and one column up, off every tile, each engine, strides, padding,
partial gradients, streams and captured graphs."""
from __future__ import annotations

import pytest
import torch

import orda_ce_kernel as orda
from tests._layers import ACTS, check, ffn64, linear64, random_inputs

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def linear_case(N, K, O, dtype, act, bias, residual, seed=0, train=True):
    shapes = {"x": ((N, K), 1.0), "w": ((O, K), K ** -0.5)}
    if bias:
        shapes["bias"] = ((O,), 0.5)
    if residual:
        shapes["residual"] = ((N, O), 1.0)
    if train:
        shapes["dy"] = ((N, O), 1.0)
    return random_inputs(shapes, dtype, seed, integers=act == "relu")


def run_linear(t, act, train=True):
    leaves = {n: v.cuda().requires_grad_(train) for n, v in t.items() if n != "dy"}
    y = orda.fused_linear(leaves["x"], leaves["w"], leaves.get("bias"), leaves.get("residual"), activation=act)
    got = {"y": y}
    if train:
        got.update(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())))
    return got


def want_linear(t, act, dtype):
    return linear64(act, dtype, **{n: v.double() for n, v in t.items()})


LINEAR_SIZES = [
    (1, 1, 1), (1, 8, 3), (2, 7, 9), (1, 300, 129), (16, 264, 100), (17, 264, 100), (33, 72, 65), (64, 64, 64),
    (100, 200, 300), (129, 1000, 257), (255, 136, 520), (300, 64, 8), (512, 33, 31), (5, 2050, 40),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", LINEAR_SIZES, ids=str)
def test_linear_sizes(size, dtype):
    t = linear_case(*size, dtype, "silu", True, True, seed=sum(size))
    check(run_linear(t, "silu"), want_linear(t, "silu", dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_linear_epilogues(act, bias, residual, dtype):
    for N, K, O in ((3, 96, 77), (90, 96, 77), (70, 128, 136)):
        t = linear_case(N, K, O, dtype, act, bias, residual, seed=N)
        check(run_linear(t, act), want_linear(t, act, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 4096, 1030), (40, 4096, 300), (600, 1024, 1100), (2100, 520, 1000), (200, 8200, 72)], ids=str)
def test_linear_larger(size, dtype):
    """Several tiles, K in ranges, the last tile of a band."""
    t = linear_case(*size, dtype, "gelu", True, True, seed=1, train=size[0] > 1)
    train = "dy" in t
    check(run_linear(t, "gelu", train), want_linear(t, "gelu", dtype))


def ffn_case(N, H, F, O, dtype, act, residual, seed=0, train=True):
    shapes = {"x": ((N, H), 1.0), "w_gate": ((F, H), H ** -0.5), "w_up": ((F, H), H ** -0.5), "w_down": ((O, F), F ** -0.5)}
    if residual:
        shapes["residual"] = ((N, O), 1.0)
    if train:
        shapes["dy"] = ((N, O), 1.0)
    return random_inputs(shapes, dtype, seed, integers=act == "relu")


def run_ffn(t, act, train=True):
    leaves = {n: v.cuda().requires_grad_(train) for n, v in t.items() if n != "dy"}
    y = orda.gated_feed_forward(leaves["x"], leaves["w_gate"], leaves["w_up"], leaves["w_down"], leaves.get("residual"),
                                activation=act)
    got = {"y": y}
    if train:
        got.update(zip(leaves, torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())))
    return got


def want_ffn(t, act, dtype):
    d = {n: v.double() for n, v in t.items()}
    return ffn64(act, dtype, d["x"], d["w_gate"], d["w_up"], d["w_down"], d.get("residual"), d.get("dy"))


FFN_SIZES = [
    (1, 1, 1, 1), (1, 8, 3, 5), (2, 7, 9, 11), (1, 300, 129, 40), (16, 264, 100, 264), (17, 264, 100, 72), (33, 72, 65, 72),
    (64, 64, 64, 64), (100, 200, 300, 200), (129, 250, 682, 250), (255, 136, 520, 130), (512, 33, 31, 17),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", FFN_SIZES, ids=str)
def test_ffn_sizes(size, dtype):
    t = ffn_case(*size, dtype, "silu", True, seed=sum(size))
    check(run_ffn(t, "silu"), want_ffn(t, "silu", dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_ffn_activations(act, dtype):
    for N, residual in ((3, True), (90, False)):
        t = ffn_case(N, 96, 200, 88, dtype, act, residual, seed=N)
        check(run_ffn(t, act), want_ffn(t, act, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(1, 1024, 2730, 1024), (50, 1024, 2730, 1024), (600, 512, 1408, 520), (2100, 264, 700, 264)], ids=str)
def test_ffn_larger(size, dtype):
    t = ffn_case(*size, dtype, "silu", False, seed=2, train=size[0] > 1)
    check(run_ffn(t, "silu", "dy" in t), want_ffn(t, "silu", dtype))


@pytest.mark.parametrize("N", [4, 200])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_inputs_are_read_in_place(dtype, N):
    """Column slices of wider tensors (aligned and not), a transposed weight, leading dimensions."""
    t = linear_case(N, 96, 136, dtype, "gelu", True, True, seed=5)
    want = want_linear(t, "gelu", dtype)
    dev = {n: v.cuda() for n, v in t.items()}
    wide = torch.full((N, 400), float("nan"), dtype=dtype, device="cuda")
    for at in (0, 16, 3):
        wide.fill_(float("nan"))
        x = wide[:, at:at + 96]
        x.copy_(dev["x"])
        r = wide[:, at + 200:at + 336]
        r.copy_(dev["residual"])
        w = dev["w"].t().contiguous().t() if at == 3 else dev["w"]
        y = orda.fused_linear(x.view(2, N // 2, 96), w, dev["bias"], r.view(2, N // 2, 136), activation="gelu")
        assert y.shape == (2, N // 2, 136)
        check({"y": y}, {"y": want["y"]})
    xs = wide[:, 16:112].detach()
    xs.copy_(dev["x"])
    xs.requires_grad_(True)
    y = orda.fused_linear(xs, dev["w"], dev["bias"], dev["residual"], activation="gelu")
    check({"x": torch.autograd.grad(y, xs, dev["dy"])[0]}, {"x": want["x"]})


@pytest.mark.parametrize("N", [4, 200])
def test_fused_weight_halves(N):
    """w_gate and w_up as two halves, and as alternate rows, of one tensor; gradients reach it."""
    t = ffn_case(N, 96, 72, 88, torch.bfloat16, "silu", False, seed=6)
    want = want_ffn(t, "silu", torch.bfloat16)
    d = {n: v.cuda() for n, v in t.items()}
    both = torch.cat([d["w_gate"], d["w_up"]]).requires_grad_(True)
    y = orda.gated_feed_forward(d["x"], both[:72], both[72:], d["w_down"])
    y.backward(d["dy"])
    check({"y": y, "w_gate": both.grad[:72], "w_up": both.grad[72:]}, {n: want[n] for n in ("y", "w_gate", "w_up")})
    mixed = torch.stack([d["w_gate"], d["w_up"]], 1).reshape(144, 96)
    check({"y": orda.gated_feed_forward(d["x"], mixed[0::2], mixed[1::2], d["w_down"])}, {"y": want["y"]})


def test_partial_gradients_and_expanded_grad_output():
    t = linear_case(90, 96, 77, torch.bfloat16, "silu", True, True, seed=7)
    t["dy"] = torch.ones_like(t["dy"])
    want = want_linear(t, "silu", torch.bfloat16)
    d = {n: v.cuda() for n, v in t.items()}
    for name in ("x", "w", "bias", "residual"):
        leaf = d[name].clone().requires_grad_(True)
        a = {**d, name: leaf}
        y = orda.fused_linear(a["x"], a["w"], a["bias"], a["residual"], activation="silu")
        y.sum().backward()  # (an expanded scalar as the gradient)
        check({name: leaf.grad}, {name: want[name]})
    f = ffn_case(90, 96, 72, 88, torch.bfloat16, "silu", True, seed=8)
    f["dy"] = torch.ones_like(f["dy"])
    want = want_ffn(f, "silu", torch.bfloat16)
    d = {n: v.cuda() for n, v in f.items()}
    for name in ("x", "w_gate", "w_up", "w_down", "residual"):
        leaf = d[name].clone().requires_grad_(True)
        a = {**d, name: leaf}
        orda.gated_feed_forward(a["x"], a["w_gate"], a["w_up"], a["w_down"], a["residual"]).sum().backward()
        check({name: leaf.grad}, {name: want[name]})


def test_retained_graph_gives_the_same_gradients_twice():
    t = ffn_case(40, 96, 72, 88, torch.bfloat16, "gelu", True, seed=9)
    leaves = {n: v.cuda().requires_grad_(True) for n, v in t.items() if n != "dy"}
    y = orda.gated_feed_forward(*[leaves[n] for n in ("x", "w_gate", "w_up", "w_down", "residual")], activation="gelu")
    one = torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda(), retain_graph=True)
    two = torch.autograd.grad(y, list(leaves.values()), t["dy"].cuda())
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_no_tokens():
    x = torch.empty(0, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(24, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = orda.fused_linear(x, w, activation="silu")
    y.sum().backward()
    assert y.shape == (0, 24) and x.grad.shape == (0, 16) and not w.grad.any()
    wd = torch.randn(8, 24, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = orda.gated_feed_forward(x, w, w, wd)
    y.sum().backward()
    assert y.shape == (0, 8) and not wd.grad.any()


@pytest.mark.parametrize("N", [2, 40, 300])
def test_infinities_and_nan_stay_in_their_rows(N):
    """A row of x with an infinity or a NaN leaves every other row as it is: the same bits in 16 bits and for few rows; in
    fp32 a tile that holds an infinity is multiplied on the native fp32 MFMA instead of as three bf16 planes, so its other
    rows round differently, and both ways are within the bound of the definition."""
    for dtype in DTYPES:
        t = linear_case(N, 96, 77, dtype, "none", True, False, seed=10, train=False)
        bad = {**t, "x": t["x"].clone()}
        bad["x"][0, 5], bad["x"][1, 7] = float("inf"), float("nan")
        clean, got = run_linear(t, "none", False)["y"], run_linear(bad, "none", False)["y"]
        want = bad["x"].double() @ bad["w"].double().t() + bad["bias"].double()
        if dtype == torch.float32 and N > 16:
            rest = {**t, "x": t["x"][2:]}
            check({"y": got[2:]}, want_linear(rest, "none", dtype))
        else:
            assert torch.equal(got[2:], clean[2:])
        assert torch.equal(got[0].isinf().cpu(), want[0].isinf()) and torch.equal(got[0].sign().cpu().double()[want[0].isinf()], want[0].sign()[want[0].isinf()])
        assert bool(got[1].isnan().all())


def test_results_do_not_depend_on_the_call(seed=11):
    """The same inputs give the same bits, whatever ran in between (no atomics, no state)."""
    t = ffn_case(200, 264, 520, 264, torch.float16, "silu", True, seed=seed)
    first = run_ffn(t, "silu")
    run_ffn(ffn_case(50, 96, 72, 88, torch.float16, "silu", True, seed=1), "silu")
    second = run_ffn(t, "silu")
    assert all(torch.equal(first[n], second[n]) for n in first)


def test_another_stream():
    t = linear_case(200, 264, 520, torch.bfloat16, "silu", True, True, seed=12)
    want = want_linear(t, "silu", torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run_linear(t, "silu")
    torch.cuda.current_stream().wait_stream(s)
    check(got, want)


@pytest.mark.parametrize("N", [3, 200])
def test_captured_forward_and_backward(N):
    """A training step of both operators captured once and replayed on new data, eager work between the replays."""
    t = ffn_case(N, 96, 200, 96, torch.bfloat16, "silu", False, seed=13)
    p = linear_case(N, 96, 72, torch.bfloat16, "gelu", True, False, seed=14)
    static = {n: v.cuda() for n, v in t.items() if n not in ("dy",)}
    static.update({"pw": p["w"].cuda(), "pb": p["bias"].cuda(), "dy": p["dy"].cuda()})
    names = ("x", "w_gate", "w_up", "w_down", "pw", "pb")

    def step():
        a = {n: static[n].detach().requires_grad_(True) for n in names}
        h = orda.gated_feed_forward(a["x"], a["w_gate"], a["w_up"], a["w_down"])
        y = orda.fused_linear(h, a["pw"], a["pb"], activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, [a[n] for n in names], static["dy"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for n in names:
            static[n].copy_(static[n][torch.randperm(static[n].shape[0], generator=g, device="cuda")])
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_a_students_step(tmp_path):
    """The operators as they are used: block, projector, loss on the projected states, backward, clipping -- against the
    same step in float64 by autograd.  Bounds: bf16 rounds 12 times on the longest way from the loss to a gradient (three
    products' operands each way, a, b, z, h, dlogits, outputs), each 2^-9 of a value; errors of independent roundings add
    up to less than their sum, so every gradient is within 12 * 2^-9 of its norm."""
    N, H, F, V = 192, 128, 344, 1000
    g = torch.Generator().manual_seed(15)
    bf = torch.bfloat16
    t = {"x": torch.randn(N, H, generator=g), "w_gate": torch.randn(F, H, generator=g) * H ** -0.5,
         "w_up": torch.randn(F, H, generator=g) * H ** -0.5, "w_down": torch.randn(H, F, generator=g) * F ** -0.5,
         "proj": torch.randn(H, H, generator=g) * H ** -0.5, "bias": torch.randn(H, generator=g) * 0.1,
         "head": torch.randn(V, H, generator=g) * H ** -0.5}
    t = {n: v.to(bf) for n, v in t.items()}
    teacher = torch.randn(N, H, generator=g).to(bf)
    labels = torch.randint(0, V, (N,), generator=g)
    dev = {n: torch.nn.Parameter(v.cuda()) for n, v in t.items()}
    y = orda.gated_feed_forward(dev["x"], dev["w_gate"], dev["w_up"], dev["w_down"], dev["x"])
    z = orda.fused_linear(y, dev["proj"], dev["bias"], activation="silu")
    out = orda.distillation_loss(z, dev["head"], labels.cuda(), orda.TiedTeacher(teacher.cuda()), kl_weight=1.0,
                                 kl_temperature=2.0, teacher_ce_weight=0.0)
    out.loss.backward()
    total = orda.clip_grad_norm_(dev.values(), 0.5)
    ref = {n: v.double().requires_grad_(True) for n, v in t.items()}
    y = torch.nn.functional.silu(ref["x"] @ ref["w_gate"].t()) * (ref["x"] @ ref["w_up"].t()) @ ref["w_down"].t() + ref["x"]
    z = torch.nn.functional.silu(y @ ref["proj"].t() + ref["bias"])
    ls, lt = z @ ref["head"].t(), (teacher.double() @ ref["head"].t()).detach()
    ps, pt = torch.log_softmax(ls / 2, -1), torch.log_softmax(lt / 2, -1)
    loss = torch.nn.functional.cross_entropy(ls, labels) + 4 * (pt.exp() * (pt - ps)).sum(-1).mean()
    loss.backward()
    norm = sum(v.grad.square().sum() for v in ref.values()).sqrt()
    tol = 12 * 2.0 ** -9
    assert abs(float(total) - float(norm)) <= tol * float(norm)
    for n, v in ref.items():
        want = v.grad * min(1.0, 0.5 / float(norm))
        assert float((dev[n].grad.double().cpu() - want).norm()) <= 2 * tol * float(want.norm()), n
