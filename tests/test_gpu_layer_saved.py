"""The projection and the feed-forward block under saved-tensor hooks: what a hook hands back (a dense copy from the host, a
copy at another alignment) is read by its own pitch, whatever the saved tensor's was."""
from __future__ import annotations

import pytest
import torch

import orda_ce_kernel as orda
from tests.test_gpu_layers import DTYPES, ffn_case, linear_case, want_ffn, want_linear
from tests._layers import check

pytestmark = pytest.mark.gpu


def apart(t, at=16):
    """The same values in rows 400 elements apart; what lies between them is NaN."""
    wide = torch.full((t.shape[0], 400), float("nan"), dtype=t.dtype, device="cuda")
    view = wide[:, at:at + t.shape[1]]
    view.copy_(t)
    return view.detach().requires_grad_(True)


def misaligned(t):
    """A dense copy one element past an aligned address."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
    return flat.view(t.shape).copy_(t)


def hooks():
    return {
        "save_on_cpu": lambda: torch.autograd.graph.save_on_cpu(),
        "misaligned": lambda: torch.autograd.graph.saved_tensors_hooks(misaligned, lambda t: t),
        "transposed": lambda: torch.autograd.graph.saved_tensors_hooks(
            lambda t: t.t().contiguous() if t.ndim == 2 else t, lambda t: t.t() if t.ndim == 2 else t),
    }


@pytest.mark.parametrize("hook", list(hooks()))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [4, 90])
def test_linear_of_row_strided_operands(N, dtype, hook):
    t = linear_case(N, 96, 136, dtype, "gelu", True, False, seed=40)
    leaves = [apart(t["x"].cuda()), apart(t["w"].cuda(), 32), t["bias"].cuda().requires_grad_(True)]
    with hooks()[hook]():
        y = orda.fused_linear(*leaves, activation="gelu")
    got = dict(zip(("x", "w", "bias"), torch.autograd.grad(y, leaves, t["dy"].cuda())))
    check({"y": y, **got}, want_linear(t, "gelu", dtype))


@pytest.mark.parametrize("hook", list(hooks()))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [4, 90])
def test_block_of_row_strided_operands(N, dtype, hook):
    t = ffn_case(N, 96, 72, 88, dtype, "silu", False, seed=41)
    names = ("x", "w_gate", "w_up", "w_down")
    leaves = [apart(t[n].cuda(), 16 * (1 + i % 2)) for i, n in enumerate(names)]
    with hooks()[hook]():
        y = orda.gated_feed_forward(*leaves)
    got = dict(zip(names, torch.autograd.grad(y, leaves, t["dy"].cuda())))
    check({"y": y, **got}, want_ffn(t, "silu", dtype))


def test_padded_operands_and_one_gate_weight_handed_back_apart():
    """Odd widths (the node saves padded copies), and a hook after which gate and up have different pitches."""
    t = ffn_case(50, 97, 73, 89, torch.bfloat16, "silu", False, seed=42)
    names = ("x", "w_gate", "w_up", "w_down")
    seen = []

    def pack(v):
        seen.append(v.shape)
        if len(seen) == 2:  # w_gate
            wide = torch.full((v.shape[0], 400), float("nan"), dtype=v.dtype, device=v.device)
            wide[:, 8:8 + v.shape[1]].copy_(v)
            return wide[:, 8:8 + v.shape[1]]
        return misaligned(v)

    leaves = [t[n].cuda().requires_grad_(True) for n in names]
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v):
        y = orda.gated_feed_forward(*leaves)
    got = dict(zip(names, torch.autograd.grad(y, leaves, t["dy"].cuda())))
    assert len(seen) == 7
    check({"y": y, **got}, want_ffn(t, "silu", torch.bfloat16))


def test_hooks_that_hand_back_another_dtype():
    """Values that a hook keeps in fp32 (or, bytes, as int32) and hands back so."""
    t = ffn_case(90, 96, 72, 88, torch.bfloat16, "silu", False, seed=43)
    names = ("x", "w_gate", "w_up", "w_down")
    leaves = [t[n].cuda().requires_grad_(True) for n in names]
    wide = lambda v: v.int() if v.dtype == torch.uint8 else v.float()  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(wide, lambda v: v):
        y = orda.gated_feed_forward(*leaves)
    check({"y": y, **dict(zip(names, torch.autograd.grad(y, leaves, t["dy"].cuda())))}, want_ffn(t, "silu", torch.bfloat16))


def test_hooks_that_hand_back_something_else_are_refused():
    x, w = (torch.randn(40, 16, device="cuda", requires_grad=True) for _ in range(2))
    for other in (lambda t: t[:-1], lambda t: t.cpu(), lambda t: t.reshape(-1)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other):
            y = orda.fused_linear(x, w)
            z = orda.gated_feed_forward(x, w, w, torch.ones(8, 40, device="cuda"))
        for v in (y, z):
            with pytest.raises(RuntimeError, match="came back from its hooks"):
                v.sum().backward()
