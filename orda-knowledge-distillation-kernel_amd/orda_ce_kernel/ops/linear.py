"""The projection: a matrix product with bias, activation and residual in its epilogue.

    y = act(x W^T + bias) + residual

One kernel computes it (few rows: one that streams W; more: tiles of the matrix cores, with K split over workgroups where
there are few tiles); for the backward pass it also keeps z = x W^T + bias where an activation needs it (fp32; for 16-bit
tensors the upper 24 bits of the fp32 values).  Backward: dz = dy act'(z) and the bias gradient in one pass over dy and z, then dx = dz W and dW = dz^T x;
the residual's gradient is dy.  Products accumulate in fp32, every output is rounded once.  No counterpart in the
reference, whose models use torch.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from .. import _native
from .._runtime import default_compute_dtype
from ._layers import (activation_torch, check_shape, check_tensors, needs_function, new_grad, operand, pitch, rows_of, trim,
                      use_kernels)

__all__ = ["FusedLinearFunction", "fused_linear"]


def _forward(x2, weight, bias, res2, act: str, dtype, keep: bool):
    """(y, operands, d, problem); d None where it is not needed."""
    xo, wo = operand(x2, dtype), operand(weight, dtype)
    if bias is not None:
        bias = bias.to(dtype).contiguous()
    if res2 is not None:
        res2 = rows_of(res2, dtype)
    O = weight.shape[0]
    p = _native.Linear(abi_version=_native.ABI_VERSION, dtype=_native.DTYPE[dtype], activation=_native.ACTIVATION[act],
                       tokens=x2.shape[0], in_features=x2.shape[1], out_features=O, ldx=pitch(xo), ldw=pitch(wo),
                       ldr=pitch(res2) if res2 is not None else 0)
    y = torch.empty((x2.shape[0], O), dtype=dtype, device=x2.device)
    d = None
    if keep and act != "none":
        d = torch.empty(_native.linear_saved_bytes(p), dtype=torch.uint8, device=x2.device)
    _native.linear_forward(p, xo, wo, bias, res2, y, d)
    return y, xo, wo, d, p


class FusedLinearFunction(torch.autograd.Function):
    """``(x [N, K], weight [O, K], bias, residual [N, O], activation)`` -> ``y [N, O]``."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation: str):
        dtype = default_compute_dtype(*[t for t in (x, weight) if t is not None])
        y, xo, wo, d, p = _forward(x, weight, bias, residual, activation, dtype, True)
        ctx.save_for_backward(xo, wo, d)
        ctx.problem, ctx.dtype = p, dtype
        ctx.given = tuple(None if t is None else (t.shape, t.dtype) for t in (x, weight, bias, residual))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        xo, wo, d = ctx.saved_tensors
        (xs, xd), (ws, wd), b, r = ctx.given
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        g_r = grad_y.to(r[1]) if r is not None and need_r else None
        g_x = g_w = g_b = None
        need_b = need_b and b is not None
        if need_x or need_w or need_b:
            dy = grad_y.to(ctx.dtype).contiguous()
            g_x = new_grad(xs[0], xs[1], ctx.dtype, dy.device) if need_x else None
            g_w = new_grad(ws[0], ws[1], ctx.dtype, dy.device) if need_w else None
            g_b = torch.empty(ws[0], dtype=ctx.dtype, device=dy.device) if need_b else None
            p = _native.Linear.from_buffer_copy(ctx.problem)
            p.ldgx = p.ldgw = new_pitch(xs[1], ctx.dtype)
            _native.linear_backward(p, xo, wo, d, dy, g_x, g_w, g_b)
        return (trim(g_x, xs[1], xs, xd), trim(g_w, ws[1], ws, wd), g_b.to(b[1]) if need_b else None, g_r, None)


def new_pitch(cols: int, dtype: torch.dtype) -> int:
    mult = 4 if dtype == torch.float32 else 8
    return cols + (-cols) % mult


@torch._dynamo.disable
def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, *, activation: str = "none", backend: str = "auto") -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` in one kernel, with its backward pass.

    ``x`` is ``(..., in_features)``, ``weight`` ``(out_features, in_features)`` (``nn.Linear``'s layout), ``bias``
    ``(out_features,)``, ``residual`` ``(..., out_features)``; ``activation`` one of ``none``, ``relu``, ``gelu``,
    ``gelu_tanh``, ``silu``, ``sigmoid``.  The result has the compute dtype of ``x`` and ``weight`` (the loss's rule: an
    active autocast dtype, else bf16 if either is, fp16, fp32).  Rows that are a multiple of 16 bytes apart are read where
    they are; odd feature counts, unaligned or transposed tensors are copied first.  Gradients for every tensor; once
    differentiable.  ``backend`` as :func:`distillation_loss` has it."""
    check_tensors("fused_linear", activation, x, weight=weight, bias=bias, residual=residual)
    if weight.ndim != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] == 0:
        raise ValueError(f"fused_linear: weight must have shape (out_features, {x.shape[-1]}), got {tuple(weight.shape)}")
    O = weight.shape[0]
    out_shape = (*x.shape[:-1], O)
    check_shape("fused_linear", "bias", bias, (O,))
    check_shape("fused_linear", "residual", residual, out_shape)
    if not use_kernels(backend, x, "fused_linear"):
        dtype = default_compute_dtype(x, weight)
        y = torch.nn.functional.linear(x.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype))
        y = activation_torch(activation, y)
        return y if residual is None else y + residual.to(dtype)
    x2 = x.reshape(-1, x.shape[-1])
    res2 = None if residual is None else residual.reshape(-1, O)
    if x2.shape[0] == 0:  # nothing to launch; torch keeps the (zero) gradients
        dtype = default_compute_dtype(x, weight)
        y = torch.nn.functional.linear(x2.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype))
        return (y if residual is None else y + res2.to(dtype)).reshape(out_shape)
    if needs_function(x, weight, bias, residual):
        y = FusedLinearFunction.apply(x2, weight, bias, res2, activation)
    else:
        y = _forward(x2, weight, bias, res2, activation, default_compute_dtype(x, weight), False)[0]
    return y if x.ndim == 2 else y.reshape(out_shape)
