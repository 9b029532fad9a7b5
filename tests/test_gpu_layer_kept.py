"""The factors that a training call keeps in 16 bits: the fp32 values rounded to nearest at 24 bits, an error of at most 2^-16
of the value to either side."""
from __future__ import annotations

import ctypes

import pytest
import torch

from orda_ce_kernel import _native

pytestmark = pytest.mark.gpu


def decoded(planes, rows, pitch):
    """[rows x pitch] fp32 values from a plane of upper halves and a plane of the next bytes."""
    n = rows * pitch
    hi, lo = planes[:2 * n].view(torch.int16).int() << 16, planes[2 * n:].int() << 8
    return (hi + lo).view(torch.float32).view(rows, pitch)


def exact_values(N, F, seed):
    """x [N x 2] and w [F x 2] of whole numbers and parts of 256 whose products and sums need up to 24 bits: exact in fp32."""
    g = torch.Generator().manual_seed(seed)
    x = torch.stack([torch.randint(1, 256, (N,), generator=g).float(), torch.randint(-15, 16, (N,), generator=g).float() / 16], 1)
    w = torch.stack([torch.randint(-255, 256, (F,), generator=g).float(), torch.randint(-15, 16, (F,), generator=g).float() / 16], 1)
    return x, w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [4, 300])
def test_factors_are_rounded_to_nearest(N, dtype):
    """activation none: the kept factors are b and a themselves."""
    H, F, O, lib = 2, 200, 8, _native.library()
    (x, wg), wu = exact_values(N, F, 1), exact_values(N, F, 2)[1]
    p = _native.FeedForward(_native.ABI_VERSION, _native.DTYPE[dtype], 0, 0, N, H, F, O, 8, 8, F, O, 8, 8, 8, F)
    pad = [torch.nn.functional.pad(t, (0, 6)).to(dtype).cuda() for t in (x, wg, wu)]
    wd = torch.zeros(O, F, dtype=dtype, device="cuda")
    pitch, n = lib.orda_ffn_inner_pitch(ctypes.byref(p)), lib.orda_ffn_saved_bytes(ctypes.byref(p))
    assert n == N * pitch * 3
    y, h = torch.empty(N, O, dtype=dtype, device="cuda"), torch.empty(N, pitch, dtype=dtype, device="cuda")
    da, db = (torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    m = lib.orda_ffn_workspace_bytes(ctypes.byref(p), 0)
    ws = torch.empty(m, dtype=torch.uint8, device="cuda")
    rc = lib.orda_ffn_forward(ctypes.byref(p), *[t.data_ptr() for t in pad], wd.data_ptr(), None, y.data_ptr(), h.data_ptr(), da.data_ptr(),
                              db.data_ptr(), ws.data_ptr(), m, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.orda_last_error()
    for planes, w in ((da, wu), (db, wg)):
        want = (x.double() @ w.double().t()).cuda()
        got = decoded(planes, N, pitch).double()
        off = got[:, :F] - want
        assert bool((off.abs() <= 2.0 ** -16 * want.abs()).all())
        assert bool((off * want.sign() > 0).any()) and bool((off * want.sign() < 0).any())  # (to either side)
        assert not got[:, F:].any()


def test_infinities_and_nan_are_kept_as_they_are():
    N, F, O, lib = 20, 64, 8, _native.library()
    for dtype in (torch.bfloat16, torch.float16):
        code = {torch.bfloat16: 0x7FFF, torch.float16: 0x7FFF}[dtype]  # (a NaN of all ones)
        x = torch.zeros(N, 8, dtype=dtype, device="cuda")
        x[:, 0] = 1.0
        x[1, 0], x[2, 0] = float("inf"), -float("inf")
        x[3, 0] = torch.tensor([code], dtype=torch.int16, device="cuda").view(dtype)[0]
        w = torch.zeros(F, 8, dtype=dtype, device="cuda")
        w[:, 0] = 1.0
        wd = torch.zeros(O, F, dtype=dtype, device="cuda")
        p = _native.FeedForward(_native.ABI_VERSION, _native.DTYPE[dtype], 0, 0, N, 1, F, O, 8, 8, F, O, 8, 8, 8, F)
        n, m = lib.orda_ffn_saved_bytes(ctypes.byref(p)), lib.orda_ffn_workspace_bytes(ctypes.byref(p), 0)
        y, h = torch.empty(N, O, dtype=dtype, device="cuda"), torch.empty(N, F, dtype=dtype, device="cuda")
        da, db = (torch.empty(n, dtype=torch.uint8, device="cuda") for _ in range(2))
        ws = torch.empty(m, dtype=torch.uint8, device="cuda")
        rc = lib.orda_ffn_forward(ctypes.byref(p), x.data_ptr(), w.data_ptr(), w.data_ptr(), wd.data_ptr(), None, y.data_ptr(), h.data_ptr(),
                                  da.data_ptr(), db.data_ptr(), ws.data_ptr(), m, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.orda_last_error()
        got = decoded(db, N, F)[:, 0].tolist()
        assert got[:3] == [1.0, float("inf"), -float("inf")] and got[3] != got[3] and got[4] == 1.0
