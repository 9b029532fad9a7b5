"""The projection's C entry points at the edge of what a launch takes."""
from __future__ import annotations

import ctypes

import pytest
import torch

from orda_ce_kernel import _native

pytestmark = pytest.mark.gpu


def test_a_sum_of_partials_of_2_to_32_threads():
    """grad_x of 8192 x 2^21 elements in two ranges of K (the weight's rows are 2^23 bytes apart, so that 72 of them pass
    2^30): the sum of the ranges' partials takes four elements a thread.  Small whole numbers, exact sums."""
    N, K, O, ld = 8192, 1 << 21, 72, 1 << 22
    bf, lib = torch.bfloat16, _native.library()
    if torch.cuda.mem_get_info()[0] < 190 << 30:
        pytest.skip("needs 175 GB of device memory")
    p = _native.Linear(_native.ABI_VERSION, 0, 0, 0, N, K, O, K, ld, O, K, K)
    plan = _native.ProductPlan()
    assert lib.orda_linear_plan(ctypes.byref(p), 1, ctypes.byref(plan)) == 0 and plan.splits == 2
    g = torch.Generator(device="cuda").manual_seed(34)
    w = torch.zeros(O, ld, dtype=bf, device="cuda")
    w[:, :K] = torch.randint(-1, 2, (O, K), generator=g, device="cuda", dtype=torch.int8)
    dy = torch.randint(-1, 2, (N, O), generator=g, device="cuda", dtype=torch.int8).to(bf)
    n = lib.orda_linear_workspace_bytes(ctypes.byref(p), 1)
    ws, gx = torch.empty(n, dtype=torch.uint8, device="cuda"), torch.full((N, K), 7.0, dtype=bf, device="cuda")
    rc = lib.orda_linear_backward(ctypes.byref(p), None, w.data_ptr(), None, dy.data_ptr(), gx.data_ptr(), None, None, ws.data_ptr(), n,
                                  torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.orda_last_error()
    for a in range(0, K, 1 << 17):
        want = dy.float() @ w[:, a:min(K, a + (1 << 17))].float()
        assert torch.equal(gx[:, a:a + (1 << 17)].float(), want)  # (magnitudes up to 72: whole numbers that bf16 holds)
