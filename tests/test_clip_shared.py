"""Clipping of a parameter that is listed more than once, into other tensors: no tensor of ``out`` is left as it was without
a word."""
from __future__ import annotations

import pytest
import torch

import orda_ce_kernel as orda

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def shared(device):
    p, q = (torch.nn.Parameter(torch.zeros(6, 4, device=device)) for _ in range(2))
    p.grad, q.grad = torch.full_like(p, 3.0), torch.full_like(q, 4.0)
    return p, q


@pytest.mark.parametrize("device", DEVICES)
def test_two_outputs_of_one_parameter_are_refused(device):
    p, q = shared(device)
    outs = [torch.full((6, 4), 7.0, device=device) for _ in range(3)]
    with pytest.raises(ValueError, match="parameters 0 and 2 are one"):
        orda.clip_grad_norm_([p, q, p], 1.0, out=outs)
    assert all(bool((o == 7).all()) for o in outs)


@pytest.mark.parametrize("device", DEVICES)
def test_one_output_of_one_parameter_is_written_once(device):
    p, q = shared(device)
    a, flat = torch.zeros(6, 4, device=device), torch.zeros(24, device=device)
    for again in (a, a.view(6, 4)):
        total = orda.clip_grad_norm_([p, q, p], 1.0, out=[a, flat.view(6, 4), again])
        norm = (24 * 25.0) ** 0.5
        assert float(total) == pytest.approx(norm, rel=1e-6)
        assert torch.allclose(a, torch.full_like(a, 3.0 / norm)) and torch.allclose(flat, torch.full_like(flat, 4.0 / norm))
    assert float(orda.clip_grad_norm_([p, q, p], 1e9)) == pytest.approx(norm, rel=1e-6)
