"""The projection: a matrix product with bias, activation and residual in its epilogue.

    y = act(x W^T + bias) + residual

One kernel computes it (few rows: one that streams W; more: tiles of the matrix cores, with K split over workgroups where
there are few tiles); for the backward pass it also keeps d = act'(x W^T + bias) where there is an activation (fp32; for
16-bit tensors rounded to the upper 24 bits).  Backward: dz = dy d and the bias gradient in one pass over dy and d,
then dx = dz W and dW = dz^T x; the residual's gradient is dy.  Products accumulate in fp32, every output is rounded once.
The operands, workspaces and the autograd node are in csrc/torch_ops.cpp.  No counterpart in the reference, whose models use
torch.
"""
from __future__ import annotations

import torch

from .. import _native
from .._runtime import default_compute_dtype
from ._layers import activation_torch, check_shape, check_tensors, needs_function, use_kernels

__all__ = ["fused_linear"]


@torch._dynamo.disable
def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, *, activation: str = "none", backend: str = "auto") -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual`` in one kernel, with its backward pass.

    ``x`` is ``(..., in_features)``, ``weight`` ``(out_features, in_features)`` (``nn.Linear``'s layout), ``bias``
    ``(out_features,)``, ``residual`` ``(..., out_features)``; ``activation`` one of ``none``, ``relu``, ``gelu``,
    ``gelu_tanh``, ``silu``, ``sigmoid``.  The result has the compute dtype of ``x`` and ``weight`` (the loss's rule: an
    active autocast dtype, else bf16 if either is, fp16, fp32).  Rows that are a multiple of 16 bytes apart are read where
    they are; odd feature counts, unaligned or transposed tensors are copied first.  Gradients for every tensor; once
    differentiable.  A training call with an activation keeps 3 bytes (fp32: 4) per output element.  ``backend`` as :func:`distillation_loss` has it."""
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
    x2 = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    res2 = residual if residual is None or residual.ndim == 2 else residual.reshape(-1, O)
    if x2.shape[0] == 0:  # nothing to launch; torch keeps the (zero) gradients
        dtype = default_compute_dtype(x, weight)
        y = torch.nn.functional.linear(x2.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype))
        return (y if residual is None else y + res2.to(dtype)).reshape(out_shape)
    y = _native.torch_ops().linear(x2, weight, bias, res2, _native.ACTIVATION[activation], default_compute_dtype(x, weight),
                                   needs_function(x, weight, bias, residual))
    return y if x.ndim == 2 else y.reshape(out_shape)
