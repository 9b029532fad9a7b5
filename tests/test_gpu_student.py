"""The embedding, dropout, layer norm and attention as programs call them: a student of them with the projection, the
feed-forward block, the loss and clipping; captured steps, streams, threads, checkpointing, saved-tensor hooks, autocast."""
from __future__ import annotations

import threading

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

import orda_ce_kernel as orda

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


# ------------------------------------------------------------------- a student
V, E, HEADS, KV, D, INNER, LAYERS = 500, 128, 4, 2, 32, 208, 2


def make(seed=0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    p = {"embed": torch.randn(V, E, generator=g) * 0.5}
    for i in range(LAYERS):
        for n, shape in (("qkv", ((HEADS + 2 * KV) * D, E)), ("o", (E, HEADS * D)), ("gate", (INNER, E)), ("up", (INNER, E)), ("down", (E, INNER))):
            p[f"{n}{i}"] = torch.randn(*shape, generator=g) * shape[1] ** -0.5
        for n in ("n1", "n2"):
            p[f"{n}{i}"], p[f"{n}b{i}"] = 1 + 0.1 * torch.randn(E, generator=g), 0.1 * torch.randn(E, generator=g)
    p["nf"], p["nfb"] = torch.ones(E), torch.zeros(E)
    p["head"] = torch.randn(V, E, generator=g) * 0.05
    # (values that 16 bits hold, so that every dtype starts from the same ones)
    return {n: v.to(BF).to(dtype).cuda().requires_grad_(True) for n, v in p.items()}


def student(p, ids, documents, seed, drop=0.1, backend="auto"):
    B, S = ids.shape
    kw = dict(backend=backend)
    x = orda.counter_dropout(orda.token_embedding(ids, p["embed"], scale=2.0, **kw), drop, seed=seed, site=99, **kw)
    stream, branch = x, None
    for i in range(LAYERS):
        if branch is None:
            y = orda.layer_norm(stream, p[f"n1{i}"], p[f"n1b{i}"], **kw)
        else:
            y, stream = orda.layer_norm(branch, p[f"n1{i}"], p[f"n1b{i}"], stream, p=drop, seed=seed, site=2 * i, **kw)
        qkv = orda.fused_linear(y, p[f"qkv{i}"], **kw).view(B, S, HEADS + 2 * KV, D)
        q, k, v = qkv.split([HEADS, KV, KV], 2)
        a = orda.masked_attention(q, k, v, documents=documents, softcap=20.0, **kw)
        branch = orda.fused_linear(a.reshape(B, S, HEADS * D), p[f"o{i}"], **kw)
        y, stream = orda.layer_norm(branch, p[f"n2{i}"], p[f"n2b{i}"], stream, p=drop, seed=seed, site=2 * i + 1, **kw)
        branch = orda.gated_feed_forward(y, p[f"gate{i}"], p[f"up{i}"], p[f"down{i}"], **kw)
    y, _ = orda.layer_norm(branch, p["nf"], p["nfb"], stream, p=drop, seed=seed, site=50, **kw)
    return y


def batch(B=2, S=75, seed=1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(V, (B, S), generator=g)
    docs = torch.zeros(B, S, dtype=torch.int32)
    docs[:, 40:] = 1
    docs[1, 60:] = -1
    ids[1, 60:] = -100
    labels = torch.where(docs >= 0, torch.randint(V, (B, S), generator=g), -100)
    return ids.cuda(), docs.cuda(), labels.cuda(), torch.randn(B * S, V, generator=g).to(BF).cuda()


def step(p, ids, docs, labels, logits, seed, backend="auto"):
    h = student(p, ids, docs, seed, backend=backend).reshape(-1, E)
    kw = dict(kl_weight=0.5, student_ce_weight=0.5, kl_temperature=2.0, backend="triton" if backend == "auto" else backend)
    out = orda.distillation_loss(h, p["head"], labels.reshape(-1), orda.PrecomputedTeacher(logits=logits.to(h.dtype)), **kw)
    return out.loss, dict(zip(p, torch.autograd.grad(out.loss, list(p.values()))))


def test_a_students_step():
    """Loss and gradients in bf16 against the same formulas in torch and fp32, where the same elements are dropped: the
    gradients agree in direction (a cosine: what bf16 leaves of a depth-2 network's gradients is within a few half steps of
    2^-8 of their norm; 0.999 stands for 4.5% of it), the loss to 1%."""
    data = batch()
    loss, grads = step(make(), *data, seed=7)
    want, exact = step(make(dtype=F), *data, seed=7, backend="torch")
    assert abs(float(loss.detach()) - float(want.detach())) < 0.01 * abs(float(want.detach()))
    for n in grads:
        a, b = grads[n].float().flatten(), exact[n].flatten()
        assert float(a @ b / (a.norm() * b.norm())) > 0.999, n
    other, _ = step(make(), *data, seed=8)
    assert float(other.detach()) != float(loss.detach())


def test_a_students_training():
    """Steps with clipping and an optimizer run; every parameter has a gradient, within the bound (that a parameter moves is
    not said: an update below half a step of bf16, 2^-9 of a norm's weight, rounds back)."""
    p = make()
    opt = torch.optim.SGD(p.values(), lr=0.1)
    data = batch()
    for s in range(3):
        _, grads = step(p, *data, seed=s)
        for n, v in p.items():
            v.grad = grads[n]
        orda.clip_grad_norm_(p.values(), 1.0)
        assert all(torch.isfinite(g).all() and g.any() for g in grads.values())
        assert float(orda.grad_norm(grads.values())) < 1.01  # (each gradient is rounded by at most 2^-8 of itself)
        opt.step()
    assert all(torch.isfinite(v).all() for v in p.values())


def test_a_captured_step():
    """Forward and backward in one graph, the seed in a tensor that the program changes between replays; every replay against
    the eager step of its seed, with eager work between."""
    ids, docs, labels, logits = batch()
    p = make()
    own = {n: v.detach().clone().requires_grad_(True) for n, v in p.items()}
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            h = student(own, ids, docs, seed)
            torch.autograd.grad(h, list(own.values())[:-1], torch.ones_like(h))
    torch.cuda.current_stream().wait_stream(side)
    del h
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = student(own, ids, docs, seed)
        grads = torch.autograd.grad(h, list(own.values())[:-1], torch.ones_like(h))
    for k in (3, 4, 3, (1 << 63) - 1):
        seed.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        want = student(p, ids, docs, k)
        eager = torch.autograd.grad(want, list(p.values())[:-1], torch.ones_like(want))
        assert torch.equal(h, want)
        assert all(torch.equal(a, b) for a, b in zip(grads, eager))


def test_a_captured_call_needs_a_seed_on_the_device():
    x = torch.ones(64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="seed= as an int64 tensor"):
            orda.counter_dropout(x, 0.5)
        y = orda.counter_dropout(x, 0.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, x)


def test_two_captured_graphs_at_once():
    """Graphs of one shape, replayed one behind the other and on two streams, share nothing."""
    t = [torch.randint(300, (5000,), device="cuda") for _ in range(2)]
    w = [torch.randn(300, 72, device="cuda").to(BF).requires_grad_(True) for _ in range(2)]
    q = [torch.randn(1, 200, 2, 64, device="cuda").to(BF).requires_grad_(True) for _ in range(2)]
    docs = torch.arange(200, device="cuda")[None] // 70

    def work(i):
        y = orda.token_embedding(t[i], w[i])
        a = orda.masked_attention(q[i], q[i], q[i], documents=docs)
        n = orda.layer_norm(y, w[i][0].detach())
        return torch.autograd.grad((n, a), (w[i], q[i]), (n.detach(), a.detach()))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(i))
        graphs.append(g)
    want = []
    for i in range(2):
        leaf_w, leaf_q = w[i].detach().requires_grad_(True), q[i].detach().requires_grad_(True)
        w[i], q[i] = leaf_w, leaf_q
        want.append(work(i))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------- each call
def calls():
    """(name, function of leaves, leaves)"""
    x, r = torch.randn(50, 72, device="cuda").to(BF), torch.randn(50, 72, device="cuda").to(BF)
    w, b = torch.randn(72, device="cuda"), torch.randn(72, device="cuda")
    ids = torch.randint(-2, 40, (50,), device="cuda")
    q, k = torch.randn(2, 90, 4, 40, device="cuda").to(BF), torch.randn(2, 90, 2, 40, device="cuda").to(BF)
    docs = torch.arange(90, device="cuda").repeat(2, 1) // 33
    return [
        ("dropout", lambda x, r: orda.counter_dropout(x, 0.3, r, seed=4), [x, r]),
        ("norm", lambda x, w, b: orda.layer_norm(x, w, b), [x, w, b]),
        ("norm with residual", lambda x, w, b, r: sum(orda.layer_norm(x, w, b, r, p=0.3, seed=4)), [x, w, b, r]),
        ("norm with residual, one dtype", lambda x, w, r: sum(orda.layer_norm(x, w, None, r)), [x, w.to(BF), r]),
        ("embedding", lambda e: orda.token_embedding(ids, e, scale=2.0), [torch.randn(40, 72, device="cuda")]),
        ("attention", lambda q, k, v: orda.masked_attention(q, k, v, documents=docs, softcap=9.0, slopes=torch.ones(4, device="cuda")), [q, k, k * 2]),
    ]


@pytest.fixture(params=range(6), ids=lambda i: ("dropout", "norm", "norm_residual", "norm_one_dtype", "embedding", "attention")[i])
def call(request):
    torch.manual_seed(request.param)
    _, f, leaves = calls()[request.param]
    return f, [v.detach().requires_grad_(True) for v in leaves]


def gradients(f, leaves, seed=3):
    y = f(*leaves)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(seed)).to(y.dtype).cuda()
    return (y.detach(), *torch.autograd.grad(y, leaves, dy))


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_differentiable_once(call):
    f, leaves = call
    (g, *_) = torch.autograd.grad(f(*leaves).float().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.float().sum().backward()


def test_forward_mode_and_transforms_are_refused(call):
    f, leaves = call
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="jvp"):
            f(forward_ad.make_dual(leaves[0].detach(), torch.ones_like(leaves[0])), *[v.detach() for v in leaves[1:]])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: f(a, *[v.detach() for v in leaves[1:]]).float().sum())(leaves[0].detach())


def test_checkpointing(call):
    f, leaves = call
    plain = gradients(f, leaves)
    assert same(plain, gradients(lambda *a: checkpoint(f, *a, use_reentrant=False), leaves))


def test_checkpointing_draws_the_same_seed():
    x = torch.randn(64, 64, device="cuda", requires_grad=True)
    y = checkpoint(lambda a: orda.counter_dropout(a, 0.5), x, use_reentrant=False)
    (g,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g > 0, y.detach() != 0)


def test_saved_tensors_on_the_host(call):
    """Offloaded and back (dense, at other addresses), and back in another dtype: the same gradients."""
    f, leaves = call
    plain = gradients(f, leaves)
    with torch.autograd.graph.save_on_cpu():
        assert same(plain, gradients(f, leaves))

    def unaligned(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
        return flat.view(t.shape).copy_(t)

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unaligned):
        assert same(plain, gradients(f, leaves))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.double() if t.is_floating_point() else t.long()):
        assert same(plain, gradients(f, leaves))


def test_saved_tensors_of_another_shape_are_refused(call):
    f, leaves = call
    saved = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t) or t, lambda t: t.reshape(-1)[:-1]):
        y = f(*leaves)
        if saved:  # (dropout with a seed from the host saves nothing)
            with pytest.raises(RuntimeError, match="hooks"):
                torch.autograd.grad(y, leaves, torch.ones_like(y))


def test_changed_operands_are_noticed():
    w = torch.ones(72, device="cuda", requires_grad=True)
    x = torch.randn(9, 72, device="cuda")
    y = orda.layer_norm(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    y = orda.counter_dropout(x.requires_grad_(True), 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_inside_compiled_code_and_inference_mode(call):
    f, leaves = call
    plain = gradients(f, leaves)
    assert same(plain, gradients(torch.compile(lambda *a: f(*a), backend="eager"), leaves))
    with torch.inference_mode():
        y = f(*leaves)
    assert torch.equal(y, plain[0]) and y.grad_fn is None and y.is_inference()


def test_other_streams(call):
    """Calls in flight on two streams give what each gives alone."""
    f, leaves = call
    plain = gradients(f, leaves)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                mine = [v.detach().requires_grad_(True) for v in leaves]
                got.append(gradients(f, mine))
        torch.cuda.synchronize()
        assert all(same(plain, g) for g in got)


def test_several_threads(call):
    f, leaves = call
    plain, failures = gradients(f, leaves), []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                mine = [v.detach().requires_grad_(True) for v in leaves]
                for _ in range(5):
                    got = gradients(f, mine)
                    torch.cuda.current_stream().synchronize()
                    assert same(plain, got)
        except BaseException as e:  # noqa: BLE001
            failures.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures[0]


def test_a_captured_backward_pass_beside_an_eager_graph(call):
    """Beside a live graph of the same leaf made on the default stream it is refused with an error, in the capture; with
    leaves of its own it runs, and every replay is the eager result."""
    f, leaves = call
    plain = gradients(f, leaves)
    eager = f(*leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own = [v.detach().requires_grad_(True) for v in leaves]
        gradients(f, own)
    torch.cuda.synchronize()
    dy = torch.randn(plain[0].shape, generator=torch.Generator().manual_seed(3)).to(plain[0].dtype).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = f(*leaves)
        with pytest.raises(RuntimeError, match="same leaf"):
            torch.autograd.grad(y, leaves, dy)
        own = [v.detach().requires_grad_(True) for v in leaves]
        z = f(*own)
        got = (z.detach(), *torch.autograd.grad(z, own, dy))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert same(got, plain)
        torch.cuda.synchronize()
    assert torch.equal(eager, plain[0])


def test_mixed_dtypes():
    """fp32 and bf16 tensors side by side: the loss's rule for the result, every gradient in its tensor's dtype."""
    x, r = torch.randn(30, 40, device="cuda", requires_grad=True), torch.randn(30, 40, device="cuda").to(BF).requires_grad_(True)
    w, b = torch.ones(40, device="cuda", dtype=BF, requires_grad=True), torch.zeros(40, device="cuda", requires_grad=True)
    y, s = orda.layer_norm(x, w, b, r, p=0.2, seed=1)
    assert y.dtype == s.dtype == BF
    assert [g.dtype for g in torch.autograd.grad((y.float().sum() + s.float().sum()), (x, r, w, b))] == [F, BF, BF, F]
    d = orda.counter_dropout(x, 0.2, r, seed=1)
    assert d.dtype == BF and [g.dtype for g in torch.autograd.grad(d.float().sum(), (x, r))] == [F, BF]
    with torch.autocast("cuda", dtype=torch.float16):
        assert orda.layer_norm(x, b).dtype == orda.counter_dropout(x, 0.5, seed=1).dtype == torch.float16
    assert orda.layer_norm(x, w).dtype == F
