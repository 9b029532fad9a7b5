"""What the docstrings of a student's operators promise beside their formulas, on the CPU."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import orda_ce_kernel as orda
from orda_ce_kernel import _native


@pytest.mark.parametrize("call", [lambda x: orda.counter_dropout(x, 0.5), lambda x: orda.layer_norm(x, x[0], None, x, p=0.5)[1]],
                         ids=["dropout", "norm"])
def test_a_drawn_seed_does_not_depend_on_the_default_device(call):
    """seed=None draws from torch's CPU generator, inside torch.device() and out of it."""
    x = torch.randn(64, 64)
    torch.manual_seed(11)
    want, state = call(x), torch.get_rng_state()
    with torch.device("meta"):
        torch.manual_seed(11)
        assert torch.equal(call(x), want)
    assert torch.equal(torch.get_rng_state(), state)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kw", [dict(), dict(causal=False, softcap=3.0), dict(prefix=torch.tensor([4, 6])), dict(slopes=torch.ones(2))],
                         ids=lambda kw: "-".join(kw) or "causal")
def test_padding_of_the_gradient_from_above_may_hold_anything(kw, bad):
    """The torch formulation: what dy holds in rows without a document reaches no gradient."""
    docs = torch.tensor([[0, 0, 0, 0, -1, -1], [-3, 1, 1, -1, 2, 2]])
    g = torch.Generator().manual_seed(4)
    leaves = [torch.randn(2, 6, 2, 4, generator=g).requires_grad_(True) for _ in range(3)]
    dy = torch.randn(2, 6, 2, 4, generator=g)
    y = orda.masked_attention(*leaves, documents=docs, **kw)
    want = torch.autograd.grad(y, leaves, torch.where((docs < 0)[:, :, None, None], 0.0, dy), retain_graph=True)
    got = torch.autograd.grad(y, leaves, torch.where((docs < 0)[:, :, None, None], bad, dy))
    assert not y[docs < 0].any()
    for a, b in zip(got, want):
        assert torch.equal(a, b) and torch.isfinite(a).all() and not a[docs < 0].any()


def test_caps_past_the_range_of_fp32():
    """A cap that no score reaches leaves the scores, one below all of them nothing of them; in between it is the formula."""
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(1, 9, 2, 4, generator=g).requires_grad_(True) for _ in range(3))
    none, mean = orda.masked_attention(q, k, v), orda.masked_attention(q, k, v, scale=0.0)
    for cap, want in ((1e39, none), (1e300, none), (1e30, none), (1e-300, mean), (1e-46, mean), (1e-30, mean)):
        y = orda.masked_attention(q, k, v, softcap=cap)
        assert torch.allclose(y, want, rtol=1e-6, atol=1e-6)
        assert all(torch.isfinite(a).all() for a in torch.autograd.grad(y.sum(), (q, k, v)))


@pytest.mark.parametrize("scale", [1e39, -1e300, math.inf, math.nan])
def test_scales_past_the_range_of_fp32_are_refused(scale):
    """As infinities in fp32 they would leave NaN everywhere."""
    q = torch.zeros(1, 3, 1, 8)
    with pytest.raises(ValueError, match="scale must be finite in fp32"):
        orda.masked_attention(q, q, q, scale=scale)
    dense = (ctypes.c_int64 * 3)(24, 8, 8)
    p = _native.Attention(abi_version=_native.ABI_VERSION, dtype=0, heads=1, kv_heads=1, head_dim=8, causal=1, batch=1, length=3, q_stride=dense,
                          k_stride=dense, v_stride=dense, g_stride=dense, documents_stride=3, scale=scale, softcap=0.0)
    lib = _native.library()
    assert lib.orda_attention_workspace_bytes(ctypes.byref(p)) == 0 and "scale must be finite in fp32" in lib.orda_last_error().decode()
    assert orda.masked_attention(q, q, q, scale=-1e38).isfinite().all()
