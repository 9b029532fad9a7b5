"""The projection, the feed-forward block and the gradient norm on the CPU: the torch formulation, every refusal of the
Python layer and of the C entry points (no kernel is launched), and the plan's limits."""
from __future__ import annotations

import ctypes
import math
import shutil
import subprocess
from array import array
from pathlib import Path

import pytest
import torch

import orda_ce_kernel as orda
from orda_ce_kernel import _native
from tests._layers import ACTS, act64, ffn64, linear64

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("act", ACTS)
def test_torch_formulation_and_its_gradients(act):
    g = torch.Generator().manual_seed(0)
    x, w, b, r = (torch.randn(*s, generator=g) for s in ((2, 3, 5), (4, 5), (4,), (2, 3, 4)))
    z = x.double() @ w.double().t() + b.double()
    want = act64(act, z)[0] + r.double()
    assert torch.allclose(orda.fused_linear(x, w, b, r, activation=act).double(), want, atol=1e-5)
    wg, wu, wd = (torch.randn(*s, generator=g) for s in ((6, 5), (6, 5), (4, 6)))
    h = act64(act, x.double() @ wg.double().t())[0] * (x.double() @ wu.double().t())
    leaf = x.clone().requires_grad_(True)
    y = orda.gated_feed_forward(leaf, wg, wu, wd, r, activation=act)
    assert torch.allclose(y.double(), h @ wd.double().t() + r.double(), atol=1e-4)
    y.sum().backward()
    assert leaf.grad.shape == x.shape


def test_derivatives_against_differences():
    """act64's derivative (what the GPU tests compare gradients with) against central differences: the cube of the step
    times the third derivative (below 10) plus the step's rounding."""
    z = torch.linspace(-6, 6, 241, dtype=torch.float64) + 0.01
    for act in ACTS:
        h = 1e-4
        diff = (act64(act, z + h)[0] - act64(act, z - h)[0]) / (2 * h)
        assert float((diff - act64(act, z)[1]).abs().max()) < 10 * h * h + 1e-10


def test_compute_dtype_and_autocast():
    x, w = torch.randn(3, 8), torch.randn(4, 8).bfloat16()
    assert orda.fused_linear(x, w).dtype == torch.bfloat16
    assert orda.fused_linear(x, w.float()).dtype == torch.float32
    assert orda.gated_feed_forward(x, w, w, torch.randn(5, 4)).dtype == torch.bfloat16


def test_clipping_in_torch():
    ps = [torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(2, 3)), torch.nn.Parameter(torch.zeros(1))]
    ps[0].grad, ps[1].grad = torch.arange(5.0), torch.ones(2, 3)
    before = [p.grad.clone() for p in ps[:2]]
    total = orda.clip_grad_norm_(iter(ps), 2.0)
    assert abs(float(total) - 6.0) < 1e-5
    assert all(torch.allclose(p.grad, b * (2.0 / 6.0)) for p, b in zip(ps, before))
    outs = [torch.empty(5, dtype=torch.float16), torch.empty(2, 3), torch.empty(1)]
    assert float(orda.clip_grad_norm_(ps, 1e9, out=outs)) == pytest.approx(2.0)
    assert torch.equal(outs[1], ps[1].grad) and outs[0].dtype == torch.float16
    assert float(orda.grad_norm([])) == 0.0 and float(orda.clip_grad_norm_([], 1.0)) == 0.0
    assert float(orda.grad_norm([torch.tensor([-3.0]), torch.tensor([2.0])], math.inf)) == 3.0
    assert float(orda.grad_norm(torch.tensor([-3.0, 2.0]), 1)) == 5.0
    with pytest.raises(RuntimeError, match="non-finite"):
        ps[0].grad = torch.tensor([math.nan] * 5)
        orda.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)


X, W = torch.zeros(3, 8), torch.zeros(4, 8)


@pytest.mark.parametrize("call,error,match", [
    (lambda: orda.fused_linear(X, W, activation="swish"), ValueError, "activation must be one of"),
    (lambda: orda.fused_linear(X, torch.zeros(4, 7)), ValueError, "weight must have shape"),
    (lambda: orda.fused_linear(X, torch.zeros(8)), ValueError, "weight must have shape"),
    (lambda: orda.fused_linear(X, torch.zeros(0, 8)), ValueError, "weight must have shape"),
    (lambda: orda.fused_linear(torch.zeros(3, 0), torch.zeros(4, 0)), ValueError, "features > 0"),
    (lambda: orda.fused_linear(X, W, torch.zeros(3)), ValueError, "bias must have shape"),
    (lambda: orda.fused_linear(X, W, None, torch.zeros(3, 5)), ValueError, "residual must have shape"),
    (lambda: orda.fused_linear(X.double(), W), ValueError, "x must be bfloat16"),
    (lambda: orda.fused_linear(X, W.long()), ValueError, "weight must be bfloat16"),
    (lambda: orda.fused_linear(X, W.to("meta")), ValueError, "weight is on meta"),
    (lambda: orda.fused_linear(X, [1.0]), TypeError, "weight must be a tensor"),
    (lambda: orda.fused_linear(X, W, backend="cuda"), ValueError, "backend must be"),
    (lambda: orda.fused_linear(X, W, backend="hip"), RuntimeError, "requires the HIP extension"),
    (lambda: orda.gated_feed_forward(X, W, torch.zeros(5, 8), torch.zeros(2, 4)), ValueError, "w_up must have shape"),
    (lambda: orda.gated_feed_forward(X, torch.zeros(4, 7), W, torch.zeros(2, 4)), ValueError, "w_gate must have shape"),
    (lambda: orda.gated_feed_forward(X, W, W, torch.zeros(2, 5)), ValueError, "w_down must have shape"),
    (lambda: orda.gated_feed_forward(X, W, W, torch.zeros(2, 4), X), ValueError, "residual must have shape"),
    (lambda: orda.gated_feed_forward(X, W, W, torch.zeros(2, 4), activation=""), ValueError, "activation must be"),
    (lambda: orda.gated_feed_forward(X, W, W, torch.zeros(2, 4), backend="triton"), RuntimeError, "requires the HIP"),
    (lambda: orda.grad_norm([X], 3.0), ValueError, "norm_type must be 1, 2 or infinity"),
    (lambda: orda.grad_norm([X, 1.0]), TypeError, "expected tensors"),
    (lambda: orda.grad_norm([X.long()]), ValueError, "must be bfloat16"),
    (lambda: orda.grad_norm([X, X.to("meta")]), ValueError, "on one device"),
    (lambda: orda.grad_norm([X.to_sparse()]), ValueError, "must be dense"),
    (lambda: orda.grad_norm([X], backend="hip"), RuntimeError, "requires the HIP"),
    (lambda: orda.clip_grad_norm_([torch.nn.Parameter(X)], -1.0), ValueError, "max_norm must be >= 0"),
    (lambda: orda.clip_grad_norm_([torch.nn.Parameter(X)], math.nan), ValueError, "max_norm must be >= 0"),
    (lambda: orda.clip_grad_norm_([torch.nn.Parameter(X)], 1.0, out=[]), ValueError, "one tensor per parameter"),
])
def test_python_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


def test_clip_refuses_outputs_and_norms_that_do_not_fit():
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="out\\[0\\]"):
        orda.clip_grad_norm_([p], 1.0, out=[torch.zeros(4)])
    with pytest.raises(ValueError, match="one-element"):
        orda.clip_grad_norm_([p], 1.0, total_norm=torch.zeros(2))


# ------------------------------------------------------------------- C ABI
def linear(**kw):
    base = dict(abi_version=_native.ABI_VERSION, dtype=0, activation=1, tokens=4, in_features=16, out_features=12, ldx=16,
                ldw=16, ldr=12, ldgx=16, ldgw=16)
    return _native.Linear(**{**base, **kw})


def ffn(**kw):
    base = dict(abi_version=_native.ABI_VERSION, dtype=0, activation=4, tokens=4, hidden=16, inner=24, out_features=16,
                ldx=16, ldw=16, ldd=24, ldr=16, ldg=16, ldgx=16, ldgw=16, ldgd=24)
    return _native.FeedForward(**{**base, **kw})


def message():
    return _native.library().orda_last_error().decode()


@pytest.mark.parametrize("kw,match", [
    (dict(abi_version=3), "abi_version"), (dict(dtype=3), "dtype"), (dict(activation=6), "activation"),
    (dict(activation=-1), "activation"), (dict(reserved=1), "reserved"), (dict(tokens=0), "tokens"),
    (dict(tokens=(1 << 30) + 1), "tokens"), (dict(in_features=0), "in_features"), (dict(out_features=1 << 23), "out_features"),
    (dict(ldx=12), "ldx"), (dict(ldx=20), "ldx"), (dict(ldw=8), "ldw"), (dict(in_features=17), "ldx"),
])
def test_linear_problems_are_refused(kw, match):
    lib = _native.library()
    assert lib.orda_linear_workspace_bytes(ctypes.byref(linear(**kw)), 0) == 0
    assert match in message()
    assert lib.orda_linear_forward(ctypes.byref(linear(**kw)), 256, 256, None, None, 256, None, 256, 1 << 30, None) == -1


@pytest.mark.parametrize("kw,match", [
    (dict(abi_version=0), "abi_version"), (dict(dtype=-1), "dtype"), (dict(activation=9), "activation"),
    (dict(tokens=-1), "tokens"), (dict(hidden=0), "hidden"), (dict(inner=0), "inner"), (dict(out_features=0), "out_features"),
    (dict(ldx=8), "ldx"), (dict(ldw=18), "ldw"), (dict(ldd=16), "ldd"), (dict(inner=25), "ldd"),
])
def test_ffn_problems_are_refused(kw, match):
    lib = _native.library()
    assert lib.orda_ffn_workspace_bytes(ctypes.byref(ffn(**kw)), 1) == 0
    assert match in message()
    assert lib.orda_ffn_inner_pitch(ctypes.byref(ffn(**kw))) == 0


def test_operands_and_workspaces_are_checked_before_any_launch():
    lib, big = _native.library(), 1 << 30
    p, f = ctypes.byref(linear()), ctypes.byref(ffn())

    def refused(rc, code, text):
        assert rc == code and text in message(), (rc, message())

    refused(lib.orda_linear_forward(None, 256, 256, None, None, 256, None, 256, big, None), -1, "NULL")
    refused(lib.orda_linear_forward(p, None, 256, None, None, 256, None, 256, big, None), -1, "required")
    refused(lib.orda_linear_forward(p, 264, 256, None, None, 256, None, 256, big, None), -1, "aligned")
    refused(lib.orda_linear_forward(ctypes.byref(linear(ldr=8)), 256, 256, None, 256, 256, None, 256, big, None), -1, "ldr")
    refused(lib.orda_linear_forward(ctypes.byref(linear(ldr=(1 << 22) + 8)), 256, 256, None, 256, 256, None, 256, big, None), -1, "ldr")
    refused(lib.orda_ffn_forward(ctypes.byref(ffn(ldr=(1 << 22) + 8)), *[256] * 5, 256, 256, None, None, 256, big, None), -1, "ldr")
    refused(lib.orda_linear_forward(p, 256, 256, None, None, 256, None, None, 0, None), -2, "workspace")
    refused(lib.orda_linear_backward(p, 256, 256, None, 256, 256, 256, None, 256, big, None), -1, "d is required")
    refused(lib.orda_linear_backward(p, 256, 256, 256, None, 256, 256, None, 256, big, None), -1, "grad_output")
    refused(lib.orda_linear_backward(p, None, 256, 256, 256, 256, 256, None, 256, big, None), -1, "needs")
    refused(lib.orda_linear_backward(ctypes.byref(linear(ldgx=8)), 256, 256, 256, 256, 256, None, None, 256, big, None), -1, "ldgx")
    refused(lib.orda_linear_backward(ctypes.byref(linear(ldgw=20)), 256, 256, 256, 256, None, 256, None, 256, big, None), -1, "ldgw")
    refused(lib.orda_linear_backward(p, 256, 256, 256, 256, 256, 256, 256, 256, 16, None), -2, "workspace")
    refused(lib.orda_ffn_forward(f, 256, 256, 256, None, None, 256, 256, None, None, 256, big, None), -1, "required")
    refused(lib.orda_ffn_forward(f, 256, 256, 256, 256, None, 256, 256, 256, None, 256, big, None), -1, "together")
    refused(lib.orda_ffn_forward(f, 256, 256, 258, 256, None, 256, 256, None, None, 256, big, None), -1, "aligned")
    refused(lib.orda_ffn_forward(f, 256, 256, 256, 256, None, 256, 256, None, None, 256, 8, None), -2, "workspace")
    refused(lib.orda_ffn_backward(f, *[256] * 7, None, *[256] * 4, 256, big, None), -1, "required")
    refused(lib.orda_ffn_backward(ctypes.byref(ffn(ldg=12)), *[256] * 12, 256, big, None), -1, "ldg")
    refused(lib.orda_ffn_backward(ctypes.byref(ffn(ldgd=16)), *[256] * 12, 256, big, None), -1, "ldgd")
    refused(lib.orda_ffn_backward(f, *[256] * 12, 256, 64, None), -2, "workspace")


def grads(*rows):
    return array("q", [v for r in rows for v in r])


@pytest.mark.parametrize("row,match", [
    ((256, 0, -1, 4, 4, 4, 0), "negative"), ((0, 0, 1, 4, 4, 4, 0), "no data"), ((256, 0, 1, 4, 4, 4, 7), "dtype"),
    ((257, 0, 1, 4, 4, 4, 0), "aligned"), ((258, 0, 1, 4, 4, 4, 2), "aligned"), ((256, 0, 2, 4, 3, 4, 0), "overlap"),
    ((256, 0, 1 << 21, 1 << 21, 1 << 21, 1 << 21, 0), "2^40"),
])
def test_gradient_tables_are_checked(row, match):
    lib, t = _native.library(), grads(row)
    assert lib.orda_grad_norm(t.buffer_info()[0], 1, 2.0, 256, 256, 1 << 20, None) == -1 and match in message()
    assert lib.orda_clip_grads(t.buffer_info()[0], 1, 256, 1.0, None) == -1 and match in message()


def test_gradient_calls_are_checked():
    lib, t = _native.library(), grads((256, 0, 1, 4, 4, 4, 0))
    a = t.buffer_info()[0]
    assert lib.orda_grad_norm(a, 1, 3.0, 256, 256, 1 << 20, None) == -1 and "norm_type" in message()
    assert lib.orda_grad_norm(a, 1, 2.0, None, 256, 1 << 20, None) == -1 and "total" in message()
    assert lib.orda_grad_norm(a, 1, 2.0, 256, 256, 16, None) == -2 and "workspace" in message()
    assert lib.orda_grad_norm(None, 1, 2.0, 256, 256, 1 << 20, None) == -1 and "table" in message()
    assert lib.orda_clip_grads(a, 1, 256, -1.0, None) == -1 and "max_norm" in message()
    assert lib.orda_clip_grads(a, 1, 256, math.nan, None) == -1 and "max_norm" in message()


@pytest.mark.parametrize("rows,ok", [
    ([(1024, 0, 1, 64, 64, 64, 0), (1088, 0, 1, 64, 64, 64, 0)], False),                    # in place, overlapping
    ([(1024, 0, 1, 64, 64, 64, 0), (1024, 0, 1, 64, 64, 64, 0)], False),                    # twice the same
    ([(1024, 4096, 1, 64, 64, 64, 2 << 32), (8192, 4100, 1, 64, 64, 64, 2 << 32)], False),  # outputs overlap
    ([(1024, 1024, 1, 64, 64, 64, 2 << 32)], False),                                        # fp32 over its own bf16
    ([(1024, 4096, 1, 64, 64, 64, 0), (4096, 8192, 1, 64, 64, 64, 0)], False),              # an output over an input
    ([(1024, 0, 8, 16, 32, 32, 0), (1056, 0, 8, 17, 32, 32, 0)], False),                    # columns that meet
])
def test_memory_that_meets_is_refused(rows, ok):
    t = grads(*rows)
    assert _native.library().orda_clip_grads(t.buffer_info()[0], len(rows), 256, 1.0, None) == -1
    assert "meet in memory" in message()


def test_clip_grad_norm_and_pad_rows_are_checked():
    lib, t = _native.library(), grads((256, 0, 1, 4, 4, 4, 0))
    a = t.buffer_info()[0]
    call = lib.orda_clip_grad_norm
    assert call(a, 1, 3.0, 1.0, 256, 256, 1 << 20, None) == -1 and "norm_type" in message()
    assert call(a, 1, 2.0, -1.0, 256, 256, 1 << 20, None) == -1 and "max_norm" in message()
    assert call(a, 1, 2.0, 1.0, None, 256, 1 << 20, None) == -1 and "total" in message()
    assert call(a, 1, 2.0, 1.0, 256, 256, 16, None) == -2 and "workspace" in message()
    assert call(None, 1, 2.0, 1.0, 256, 256, 1 << 20, None) == -1 and "table" in message()
    twice = grads((1024, 0, 1, 64, 64, 64, 0), (1024, 0, 1, 64, 64, 64, 0))
    assert call(twice.buffer_info()[0], 2, 2.0, 1.0, 256, 256, 1 << 20, None) == -1 and "meet in memory" in message()

    def rows(*r):
        return (_native.Rows * len(r))(*(_native.Rows(*v) for v in r))

    good = (256, 512, 2, 5, 5, 8)
    for dtype, table, n, text in (
            (3, rows(good), 1, "dtype"), (0, rows(good), 5, "n must be"), (0, None, 1, "n must be"), (0, rows(good), -1, "n must be"),
            (0, rows((256, 520, 2, 5, 5, 8)), 1, "aligned"), (0, rows((257, 512, 2, 5, 5, 8)), 1, "aligned"),
            (0, rows((None, 512, 2, 5, 5, 8)), 1, "aligned"), (0, rows((256, 512, 2, 9, 9, 8)), 1, "pitch"),
            (0, rows((256, 512, 2, 5, 4, 8)), 1, "pitch"), (2, rows((256, 512, 2, 5, 5, 6)), 1, "pitch"),
            (0, rows((256, 512, -1, 5, 5, 8)), 1, "size"), (0, rows((256, 512, 2, 0, 5, 8)), 1, "size")):
        assert lib.orda_pad_rows(dtype, table, n, None) == -1 and text in message(), text
    assert lib.orda_pad_rows(0, None, 0, None) == 0


@pytest.mark.parametrize("tokens,ldx", [(1 << 20, 4096), (1 << 22, 16), (1000, 1 << 22), (1 << 30, 1 << 12)])
def test_long_operands_are_read_in_ranges_of_at_most_2_to_30_bytes(tokens, ldx):
    """The weight gradient's operands have tokens as K: as many ranges of it, each with its fp32 partials in the workspace."""
    p = linear(tokens=tokens, activation=0, ldx=ldx)
    n = _native.library().orda_linear_workspace_bytes(ctypes.byref(p), 1)
    dz = tokens * 16 * 2
    ranges = -(-tokens * ldx * 2 // (1 << 30))
    assert n >= dz + (ranges if ranges > 1 else 0) * 12 * 16 * 4


def test_gradients_of_the_definitions_against_differences():
    """linear64 and ffn64 (what the GPU tests compare with): the gradients' products with random directions against central
    differences of y . dy; the truncation is below h^2 times the third derivative along the direction (below 1e4 here)."""
    g = torch.Generator().manual_seed(3)

    def compare(value, grads, tensors):
        h = 1e-5
        for name, t in tensors.items():
            d = torch.randn(t.shape, generator=g, dtype=torch.float64)
            hi, lo = value({**tensors, name: t + h * d}), value({**tensors, name: t - h * d})
            assert abs(float(hi - lo) / (2 * h) - float((grads[name][0] * d).sum())) < 1e4 * h * h + 1e-7, name

    def tensors(**shapes):
        return {n: torch.randn(*s, generator=g, dtype=torch.float64) * 0.5 for n, s in shapes.items()}

    for act in ("none", "gelu", "gelu_tanh", "silu", "sigmoid"):
        t = tensors(x=(5, 7), w=(4, 7), bias=(4,), residual=(5, 4))
        dy = torch.randn(5, 4, generator=g, dtype=torch.float64)
        compare(lambda a: (linear64(act, torch.float32, **a)["y"][0] * dy).sum(), linear64(act, torch.float32, **t, dy=dy), t)
        f = tensors(x=(5, 7), w_gate=(6, 7), w_up=(6, 7), w_down=(4, 6), residual=(5, 4))

        def ffn_of(a, dy=None):
            return ffn64(act, torch.float32, a["x"], a["w_gate"], a["w_up"], a["w_down"], a["residual"], dy)

        compare(lambda a: (ffn_of(a)["y"][0] * dy).sum(), ffn_of(f, dy), f)


def _sharded_clip(rank, path, results):
    torch.distributed.init_process_group("gloo", init_method=f"file://{path}", rank=rank, world_size=2)
    g = torch.Generator().manual_seed(rank)
    p = torch.nn.Parameter(torch.zeros(1000))
    p.grad = torch.randn(1000, generator=g)
    total = orda.grad_norm([p.grad]) ** 2
    torch.distributed.all_reduce(total)
    got = orda.clip_grad_norm_([p], 0.5, total_norm=total.sqrt())
    torch.save((got, p.grad), f"{results}/{rank}")
    torch.distributed.destroy_process_group()


def test_norm_of_gradients_sharded_over_two_ranks(tmp_path):
    torch.multiprocessing.spawn(_sharded_clip, (str(tmp_path / "rendezvous"), str(tmp_path)), nprocs=2)
    shards = [torch.randn(1000, generator=torch.Generator().manual_seed(r)) for r in range(2)]
    norm = torch.cat(shards).double().norm()
    for r, s in enumerate(shards):
        got, grad = torch.load(tmp_path / str(r), weights_only=True)
        assert float(got) == pytest.approx(float(norm), rel=1e-6)
        assert torch.allclose(grad.double(), s.double() * 0.5 / norm, rtol=1e-6, atol=0)


def test_a_missing_binding_is_an_error(monkeypatch, tmp_path):
    monkeypatch.setattr(_native, "_TORCH_OPS", None)
    monkeypatch.setattr(_native, "__file__", str(tmp_path / "_native.py"))
    with pytest.raises(RuntimeError, match="orda_torch.so not found"):
        _native.torch_ops()


def test_struct_layouts_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("no gcc")
    names = {"orda_linear_t": _native.Linear, "orda_ffn_t": _native.FeedForward, "orda_rows_t": _native.Rows}
    lines = [f'printf("{t}.{f} %zu\\n", offsetof({t}, {f}));' for t, c in names.items() for f, _ in c._fields_]
    lines += [f'printf("{t} %zu\\n", sizeof({t}));' for t in names]
    lines += [f'printf("orda_grad_t.{f} %zu\\n", offsetof(orda_grad_t, {f}));'
              for f in ("data", "out", "rows", "cols", "ld", "ld_out", "dtype", "out_dtype")]
    lines.append('printf("orda_grad_t %zu\\n", sizeof(orda_grad_t));')
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "orda_ce.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "probe"
    subprocess.run([gcc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for t, c in names.items():
        assert int(got[t]) == ctypes.sizeof(c)
        assert all(int(got[f"{t}.{f}"]) == getattr(c, f).offset for f, _ in c._fields_)
    assert int(got["orda_grad_t"]) == 8 * _native.GRAD_WORDS
    assert [int(got[f"orda_grad_t.{f}"]) for f in ("data", "out", "rows", "cols", "ld", "ld_out", "dtype", "out_dtype")] == [
        0, 8, 16, 24, 32, 40, 48, 52]


def test_every_activation_has_a_code_in_the_header():
    text = (ROOT / "include" / "orda_ce.h").read_text()
    for name, code in _native.ACTIVATION.items():
        assert f"ORDA_ACT_{name.upper()} = {code}" in text
