"""Gradient norm and clipping on the GPU against float64: dtypes mixed, odd sizes and offsets, row-strided and other views,
many tensors, non-finite values, captured graphs.  Bounds: the norm is summed in fp64 and rounded once to fp32 (2^-24; the
root and the sum leave far less); a factor is a quotient of two rounded fp32 values (2^-24 each) and rounded, a clipped value
one fp32 product and one rounding to its dtype."""
from __future__ import annotations

import math

import pytest
import torch

import orda_ce_kernel as orda

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def norm64(tensors, p):
    flat = torch.cat([t.detach().double().cpu().reshape(-1) for t in tensors])
    return float(torch.linalg.vector_norm(flat, p)) if flat.numel() else 0.0


def params_of(grads):
    out = []
    for g in grads:
        p = torch.empty(g.shape, dtype=g.dtype, device=g.device)
        p.grad = g
        out.append(p)
    return out


def check_norm(total, tensors, p):
    want = norm64(tensors, p)
    assert total.dtype == torch.float32 and total.shape == ()
    assert abs(float(total) - want) <= 2.0 ** -23 * want


def check_clipped(got, before, total, max_norm):
    f = min(1.0, max_norm / (total + 1e-6))
    for g, b in zip(got, before):
        want = b.double().cpu() * f
        u = torch.finfo(g.dtype).eps / 2
        sub = torch.finfo(g.dtype).smallest_normal * torch.finfo(g.dtype).eps / 2
        assert bool(((g.double().cpu() - want).abs() <= (u + 2.0 ** -22) * want.abs() + sub).all())


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_of_flat_views(dtype, p):
    """Tensors one behind the other in a buffer, at every alignment, sizes around the 16-byte and chunk borders."""
    sizes = [1, 2, 3, 7, 8, 9, 15, 16, 17, 255, 2047, 2048, 2049, 4100, 16383, 1, 70001, 5]
    g = torch.Generator(device="cuda").manual_seed(1)
    flat = torch.randn(sum(sizes) + 4, generator=g, device="cuda").to(dtype)
    views = list(flat[3:3 + sum(sizes)].split(sizes))
    check_norm(orda.grad_norm(views, p), views, p)
    for v in views[:8]:
        check_norm(orda.grad_norm(v, p), [v], p)


@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("out", ["in_place", "bfloat16", "float16", "float32"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_clipping(dtype, out, max_norm):
    sizes = [1, 3, 8, 17, 2049, 5000, 33]
    g = torch.Generator(device="cuda").manual_seed(2)
    flat = torch.randn(sum(sizes) + 8, generator=g, device="cuda").to(dtype)
    grads = list(flat[1:1 + sum(sizes)].split(sizes))
    before, rest = [x.clone() for x in grads], flat.clone()
    dst = flat_out = None
    if out != "in_place":
        flat_out = torch.full((sum(sizes) + 8,), 7.0, dtype=getattr(torch, out), device="cuda")
        dst = list(flat_out[3:3 + sum(sizes)].split(sizes))
    total = orda.clip_grad_norm_(params_of(grads), max_norm, out=dst)
    check_norm(total, before, 2.0)
    check_clipped(grads if dst is None else dst, before, float(total), max_norm)
    if dst is None:  # (elements around the tensors stay as they were)
        assert torch.equal(flat[:1], rest[:1]) and torch.equal(flat[1 + sum(sizes):], rest[1 + sum(sizes):])
    else:
        assert torch.equal(flat, rest)
        assert bool((flat_out[:3] == 7).all()) and bool((flat_out[3 + sum(sizes):] == 7).all())


def test_mixed_dtypes_strides_and_many_tensors():
    g = torch.Generator(device="cuda").manual_seed(3)
    grads = []
    for i in range(250):  # (more than a launch's table, in every dtype)
        grads.append((torch.randn(1 + 37 * i % 401, generator=g, device="cuda") * 2.0 ** (i % 9)).to(DTYPES[i % 3]))
    wide = torch.randn(70, 50, generator=g, device="cuda").to(torch.bfloat16)
    keep = wide.clone()
    grads += [wide[:, :21], wide[:, 21:44]]                                       # two halves of one buffer, row-strided
    grads.append(torch.randn(40, 30, generator=g, device="cuda").t())             # transposed
    grads.append(torch.randn(9, 10, 12, generator=g, device="cuda")[:, ::2, 1:])  # no rows to walk
    grads.append(torch.empty(0, 5, device="cuda"))
    before = [x.clone() for x in grads]
    total = orda.clip_grad_norm_(params_of(grads), 3.0)
    check_norm(total, before, 2.0)
    check_clipped(grads, before, float(total), 3.0)
    assert torch.equal(wide[:, 44:], keep[:, 44:])


def test_out_of_row_strided_gradients():
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn(33, 40, generator=g, device="cuda").half()
    grads = [wide[:, :24], torch.randn(33, 24, generator=g, device="cuda")]
    outs = [torch.empty(33, 24, device="cuda"), torch.zeros(33, 64, device="cuda")[:, 8:32]]
    before = [x.clone() for x in grads]
    total = orda.clip_grad_norm_(params_of(grads), 1.0, out=outs)
    check_clipped(outs, before, float(total), 1.0)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))


def test_large_and_tiny_values_and_total_norm():
    """Squares beyond fp32's range in either direction; a norm from elsewhere; a shared parameter counted once."""
    for v in (1e30, 1e-30):
        x = torch.full((1000,), v, device="cuda")
        check_norm(orda.grad_norm([x]), [x], 2.0)
    x = torch.randn(100, device="cuda")
    p = params_of([x])[0]
    before = x.clone()
    check_norm(orda.clip_grad_norm_([p, p], 1e9), [before], 2.0)
    given = torch.tensor([50.0], device="cuda", dtype=torch.float64)
    assert float(orda.clip_grad_norm_([p], 5.0, total_norm=given)) == 50.0
    check_clipped([x], [before], 50.0, 5.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_non_finite_values(dtype, p):
    for bad in (math.inf, math.nan):
        grads = [torch.ones(3000, device="cuda", dtype=dtype), torch.ones(7, device="cuda", dtype=dtype)]
        grads[0][2900] = bad
        total = orda.grad_norm(grads, p)
        assert bool(total.isnan()) if math.isnan(bad) else bool(total.isinf())
        with pytest.raises(RuntimeError, match="non-finite"):
            orda.clip_grad_norm_(params_of(grads), 1.0, p, error_if_nonfinite=True)
        assert float(grads[1][0]) == 1.0
        orda.clip_grad_norm_(params_of(grads), 1.0, p)
        want = [x * torch.tensor(1.0 / (bad + 1e-6)) for x in (torch.ones(1), torch.tensor([bad]))]
        assert torch.equal(grads[1][:1].float().cpu().isnan(), want[0].isnan())
        assert bool(grads[0][2900].isnan())


def test_memory_that_meets_is_refused():
    x = torch.zeros(100, device="cuda")
    a, b = params_of([x[:60], x[40:]])
    with pytest.raises(ValueError, match="meet in memory"):
        orda.clip_grad_norm_([a, b], 1.0)
    with pytest.raises(ValueError, match="meet in memory"):
        orda.clip_grad_norm_([params_of([x[:60]])[0]], 1.0, out=[x[20:80]])
    assert float(orda.grad_norm([x[:60], x[40:]])) == 0.0


def test_captured_norm_and_clipping():
    g = torch.Generator(device="cuda").manual_seed(5)
    grads = [torch.randn(n, generator=g, device="cuda").bfloat16() for n in (100, 5000, 7)]
    fresh = [x.clone() for x in grads]
    outs = [torch.empty(x.shape, device="cuda") for x in grads]
    params = params_of(grads)
    orda.clip_grad_norm_(params, 1.0, out=outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = orda.clip_grad_norm_(params, 1.0, out=outs)
    for k in range(3):
        for x, f in zip(grads, fresh):
            x.copy_(f * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        check_norm(total, grads, 2.0)
        check_clipped(outs, grads, float(total), 1.0)
        orda.grad_norm(grads)
        torch.cuda.synchronize()


def test_more_than_2_to_31_elements():
    """One gradient past 32-bit indexes, beside a small one: 0.5 and, at its end, -3; every square and sum is exact."""
    n = (1 << 31) + 77
    big, small = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device="cuda")), torch.nn.Parameter(torch.zeros(5, device="cuda"))
    big.grad, small.grad = torch.full_like(big.data, 0.5), torch.ones(5, device="cuda")
    big.grad[-3:] = -3.0
    want = math.sqrt((n - 3) * 0.25 + 27 + 5)
    assert float(orda.grad_norm([big.grad, small.grad])) == pytest.approx(want, rel=2.0 ** -23)
    total = orda.clip_grad_norm_([big, small], want / 2)
    assert float(total) == pytest.approx(want, rel=2.0 ** -23)
    assert bool((big.grad[:-3] == 0.25).all()) and big.grad[-3:].tolist() == [-1.5] * 3
    assert torch.allclose(small.grad, torch.full_like(small.grad, 0.5), rtol=1e-5)


@pytest.mark.parametrize("n", [79, 80, 81, 320, 321, 700])
def test_tables_of_many_tensors(n):
    """As many tensors as one launch takes, one more, several launches; captured and replayed."""
    g = torch.Generator(device="cuda").manual_seed(6)
    sizes = [1 + (i * 37) % 211 for i in range(n)] + [5000]
    grads = [torch.randn(k, generator=g, device="cuda").bfloat16() for k in sizes]
    grads += [torch.randn(3 + k, generator=g, device="cuda") for k in range(0, n, 7)]
    for p in (1.0, 2.0, math.inf):
        check_norm(orda.grad_norm(grads, p), grads, p)
    params, outs = params_of(grads), [torch.empty(x.shape, device="cuda") for x in grads]
    total = orda.clip_grad_norm_(params, 0.5, out=outs)
    check_norm(total, grads, 2.0)
    check_clipped(outs, grads, float(total), 0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        total = orda.clip_grad_norm_(params, 0.5, out=outs)
    for k in range(2):
        for x in grads:
            x.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        check_norm(total, grads, 2.0)
        check_clipped(outs, grads, float(total), 0.5)
