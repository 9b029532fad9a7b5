"""Where gradients of odd widths lie: dense through the public functions, so that accumulating them into a leaf copies
nothing; through the C entry points dense or in padded rows."""
from __future__ import annotations

import ctypes

import pytest
import torch

import orda_ce_kernel as orda
from orda_ce_kernel import _native
from tests._layers import check, linear64
from tests.test_gpu_layers import DTYPES, ffn_case, linear_case, run_ffn, run_linear, want_ffn, want_linear

pytestmark = pytest.mark.gpu


def is_dense(t):
    return t.is_contiguous() and t.untyped_storage().nbytes() == t.numel() * t.element_size()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [(5, 17, 9), (90, 97, 77), (333, 1001, 203)], ids=str)
def test_gradients_are_dense(size, dtype):
    t = linear_case(*size, dtype, "silu", True, False, seed=50)
    got = run_linear(t, "silu")
    assert all(is_dense(got[n]) for n in ("x", "w", "bias"))
    check(got, want_linear(t, "silu", dtype))
    f = ffn_case(*size, 31, dtype, "silu", False, seed=51)
    got = run_ffn(f, "silu")
    assert all(is_dense(got[n]) for n in ("x", "w_gate", "w_up", "w_down"))
    check(got, want_ffn(f, "silu", dtype))
    leaf = f["w_up"].cuda().requires_grad_(True)
    for k in range(2):  # (accumulated in place the second time)
        orda.gated_feed_forward(f["x"].cuda(), f["w_gate"].cuda(), leaf, f["w_down"].cuda()).backward(f["dy"].cuda())
        assert is_dense(leaf.grad)
        if k == 0:
            assert torch.equal(leaf.grad, got["w_up"])
            first = leaf.grad.clone()
    assert torch.equal(leaf.grad, first + first)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [5, 90])
def test_pitches_of_the_c_entry_point(dtype, N):
    """grad_x and grad_weight dense, and in padded rows: the padding is written with zeros, what lies behind it stays."""
    K, O, g = 97, 77, 4 if dtype == torch.float32 else 8
    kp = -(-K // g) * g
    t = linear_case(N, K, O, dtype, "none", False, False, seed=52)
    want = linear64("none", dtype, **{n: v.double() for n, v in t.items()})
    x, w = (torch.nn.functional.pad(t[n], (0, kp - K)).cuda() for n in ("x", "w"))
    dy, lib = t["dy"].cuda(), _native.library()
    for ld in (K, kp, kp + 2 * g):
        p = _native.Linear(_native.ABI_VERSION, _native.DTYPE[dtype], 0, 0, N, K, O, kp, kp, O, ld, ld)
        n = lib.orda_linear_workspace_bytes(ctypes.byref(p), 1)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        gx, gw = (torch.full((r, ld), 7.0, dtype=dtype, device="cuda") for r in (N, O))
        rc = lib.orda_linear_backward(ctypes.byref(p), x.data_ptr(), w.data_ptr(), None, dy.data_ptr(), gx.data_ptr(), gw.data_ptr(), None,
                                      ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.orda_last_error()
        check({"x": gx[:, :K], "w": gw[:, :K]}, {m: want[m] for m in ("x", "w")})
        for v in (gx, gw):
            if ld > K:
                assert not v[:, K:kp].any() and bool((v[:, kp:] == 7).all())
    bad = _native.Linear(_native.ABI_VERSION, _native.DTYPE[dtype], 0, 0, N, K, O, kp, kp, O, K + 1, kp)
    assert lib.orda_linear_backward(ctypes.byref(bad), 256, 256, None, 256, 256, None, None, 256, 1 << 40, None) == -1
