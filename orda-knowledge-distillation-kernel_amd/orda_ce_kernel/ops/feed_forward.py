"""The gated feed-forward block.

    a = x Wg^T    b = x Wu^T    h = act(a) b    y = h Wd^T + residual

Two launches forward: both projections, the activation and the product in one kernel (a tile holds the same columns of Wg
and Wu, so a lane has a's and b's element side by side), then the down projection with the residual in its epilogue.
A training call also keeps the factors p = b act'(a) and q = act(a).  Backward, with dh = dy Wd never leaving the accumulators:

    da = dh p    db = dh q                                     (epilogue of dh's product)
    dx = da Wg + db Wu   (one product over both weights)
    dWg = da^T x    dWu = db^T x    dWd = dy^T h

h, da and db are rounded to the compute dtype as operands of the next product; p and q are kept in fp32, for 16-bit tensors
in its upper 24 bits; products accumulate in fp32.  No counterpart in the reference, whose models use torch.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from .._runtime import default_compute_dtype
from ._layers import (activation_torch, check_shape, check_tensors, needs_function, new_grad, operand, pitch, rows_of,
                      same_pitch, trim, use_kernels)

__all__ = ["GatedFeedForwardFunction", "gated_feed_forward"]


def _forward(x2, w_gate, w_up, w_down, res2, act: str, dtype, keep: bool):
    xo, dn = operand(x2, dtype), operand(w_down, dtype)
    ga, up = same_pitch(operand(w_gate, dtype), operand(w_up, dtype))
    if res2 is not None:
        res2 = rows_of(res2, dtype)
    N, O = x2.shape[0], w_down.shape[0]
    p = _native.FeedForward(abi_version=_native.ABI_VERSION, dtype=_native.DTYPE[dtype],
                            activation=_native.ACTIVATION[act], tokens=N, hidden=x2.shape[1], inner=w_gate.shape[0],
                            out_features=O, ldx=pitch(xo), ldw=pitch(ga), ldd=pitch(dn),
                            ldr=pitch(res2) if res2 is not None else 0)
    fp = _native.ffn_inner_pitch(p)
    y = torch.empty((N, O), dtype=dtype, device=x2.device)
    h = torch.empty((N, fp), dtype=dtype, device=x2.device)
    fa = fb = None
    if keep:
        n = _native.ffn_saved_bytes(p)
        fa, fb = (torch.empty(n, dtype=torch.uint8, device=x2.device) for _ in range(2))
    _native.ffn_forward(p, xo, ga, up, dn, res2, y, h, fa, fb)
    return y, (xo, ga, up, dn, h, fa, fb), p


class GatedFeedForwardFunction(torch.autograd.Function):
    """``(x [N, H], w_gate [F, H], w_up [F, H], w_down [O, F], residual [N, O], activation)`` -> ``y [N, O]``."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, residual, activation: str):
        dtype = default_compute_dtype(x, w_gate, w_up, w_down)
        y, saved, p = _forward(x, w_gate, w_up, w_down, residual, activation, dtype, True)
        ctx.save_for_backward(*saved)
        ctx.problem, ctx.dtype = p, dtype
        ctx.given = tuple(None if t is None else (t.shape, t.dtype) for t in (x, w_gate, w_up, w_down, residual))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        xo, ga, up, dn, h, fa, fb = ctx.saved_tensors
        given, need = ctx.given, ctx.needs_input_grad
        g_r = grad_y.to(given[4][1]) if given[4] is not None and need[4] else None
        grads = [None] * 4
        if any(need[:4]):
            dy = operand(grad_y, ctx.dtype)
            grads = [new_grad(*g[0], ctx.dtype, dy.device) if n else None for g, n in zip(given, need[:4])]
            p = _native.FeedForward.from_buffer_copy(ctx.problem)
            p.ldg = pitch(dy)
            mult = 4 if ctx.dtype == torch.float32 else 8
            p.ldgx = p.ldgw = p.hidden + (-p.hidden) % mult
            p.ldgd = p.inner + (-p.inner) % mult
            _native.ffn_backward(p, xo, ga, up, dn, h, fa, fb, dy, *grads)
        return (*[trim(v, g[0][1], g[0], g[1]) for v, g in zip(grads, given)], g_r, None)


@torch._dynamo.disable
def gated_feed_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
                       residual: torch.Tensor | None = None, *, activation: str = "silu",
                       backend: str = "auto") -> torch.Tensor:
    """``(activation(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T + residual``, with its backward pass.

    ``x`` is ``(..., hidden)``, ``w_gate`` and ``w_up`` ``(inner, hidden)`` (two halves of one tensor serve), ``w_down``
    ``(out_features, inner)``, ``residual`` ``(..., out_features)``; ``activation`` one of ``none``, ``relu``, ``gelu``,
    ``gelu_tanh``, ``silu``, ``sigmoid``.  Dtypes, strides, alignment and ``backend`` as :func:`fused_linear`.  A training
    call keeps h and two factors for its backward pass: 8 bytes (fp32: 12) per token and inner column."""
    check_tensors("gated_feed_forward", activation, x, w_gate=w_gate, w_up=w_up, w_down=w_down, residual=residual)
    if w_gate.ndim != 2 or w_gate.shape[1] != x.shape[-1] or w_gate.shape[0] == 0:
        raise ValueError(f"gated_feed_forward: w_gate must have shape (inner, {x.shape[-1]}), got {tuple(w_gate.shape)}")
    check_shape("gated_feed_forward", "w_up", w_up, w_gate.shape)
    if w_down.ndim != 2 or w_down.shape[1] != w_gate.shape[0] or w_down.shape[0] == 0:
        raise ValueError(f"gated_feed_forward: w_down must have shape (out_features, {w_gate.shape[0]}), "
                         f"got {tuple(w_down.shape)}")
    out_shape = (*x.shape[:-1], w_down.shape[0])
    check_shape("gated_feed_forward", "residual", residual, out_shape)
    kernels = use_kernels(backend, x, "gated_feed_forward")
    dtype = default_compute_dtype(x, w_gate, w_up, w_down)
    if not kernels or x.numel() == 0:  # (no rows: nothing to launch; torch keeps the zero gradients)
        xc = x.to(dtype)
        lin = torch.nn.functional.linear
        y = lin(activation_torch(activation, lin(xc, w_gate.to(dtype))) * lin(xc, w_up.to(dtype)), w_down.to(dtype))
        return y if residual is None else y + residual.to(dtype)
    x2 = x.reshape(-1, x.shape[-1])
    res2 = None if residual is None else residual.reshape(-1, w_down.shape[0])
    if needs_function(x, w_gate, w_up, w_down, residual):
        y = GatedFeedForwardFunction.apply(x2, w_gate, w_up, w_down, res2, activation)
    else:
        y = _forward(x2, w_gate, w_up, w_down, res2, activation, dtype, False)[0]
    return y if x.ndim == 2 else y.reshape(out_shape)
