"""The gated feed-forward block.

    a = x Wg^T    b = x Wu^T    h = act(a) b    y = h Wd^T + residual

Two launches forward: both projections, the activation and the product in one kernel (a tile holds the same columns of Wg
and Wu, so a lane has a's and b's element side by side), then the down projection with the residual in its epilogue.
A training call also keeps the factors p = b act'(a) and q = act(a).  Backward, with dh = dy Wd never leaving the accumulators:

    da = dh p    db = dh q                                     (epilogue of dh's product)
    dx = da Wg + db Wu   (one product over both weights)
    dWg = da^T x    dWu = db^T x    dWd = dy^T h

h, da and db are rounded to the compute dtype as operands of the next product; p and q are kept in fp32, for 16-bit tensors
rounded to its upper 24 bits; products accumulate in fp32.  The operands, workspaces and the autograd node are in
csrc/torch_ops.cpp.  No counterpart in the reference, whose models use torch.
"""
from __future__ import annotations

import torch

from .. import _native
from .._runtime import default_compute_dtype
from ._layers import activation_torch, check_shape, check_tensors, needs_function, use_kernels

__all__ = ["gated_feed_forward"]


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
    x2 = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    res2 = residual if residual is None or residual.ndim == 2 else residual.reshape(-1, w_down.shape[0])
    y = _native.torch_ops().feed_forward(x2, w_gate, w_up, w_down, res2, _native.ACTIVATION[activation], dtype,
                                         needs_function(x, w_gate, w_up, w_down, residual))
    return y if x.ndim == 2 else y.reshape(out_shape)
