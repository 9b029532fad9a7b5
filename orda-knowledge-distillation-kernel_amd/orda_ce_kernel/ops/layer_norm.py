"""The layer norm, with the dropout and the residual that stand in front of it in a layer.

    s = residual + dropout(x)      h = (s - mean) / sqrt(variance + eps)      y = h w + b
    g = dy w      ds' = ds + rstd (g - mean(g) - h mean(g h))      dx = dropout'(ds')      dresidual = ds'
    dw = sum of dy h      db = sum of dy

One kernel forward, two backward (the second adds up dw's and db's partial sums, in order); csrc/rownorm.hip.  y is computed
from s in fp32.  The backward pass reads s as it was written, rounded, with the row's mean and rstd in fp32; for fp32
parameters beside 16-bit activations it computes s again from x and the residual, so that their gradients have fp32's
precision.  No counterpart in the reference, whose models use torch (its student's RMS norm stands inside the loss:
StudentRMSNorm).
"""
from __future__ import annotations

import math

import torch

from .. import _native
from .._runtime import default_compute_dtype
from ._layers import check_shape, check_tensors, needs_function, use_kernels
from ._random import check_dropout, kept_factors

__all__ = ["layer_norm"]


def _torch(x, weight, bias, residual, eps, p, seed, seed_tensor, site, dtype):
    s = x.to(dtype).float()
    if p > 0.0:
        keep = kept_factors(x.shape, p, seed, seed_tensor, site, x.device)
        s = torch.where(keep > 0, s * keep, 0.0)
    if residual is not None:
        s = s + residual.to(dtype).float()
    d = s - s.mean(-1, keepdim=True)
    y = d * torch.rsqrt((d * d).mean(-1, keepdim=True) + eps) * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(dtype) if residual is None else (y.to(dtype), s.to(dtype))


@torch._dynamo.disable
def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
               *, eps: float = 1e-5, p: float = 0.0, seed: int | torch.Tensor | None = None, site: int = 0,
               backend: str = "auto"):
    """The layer norm of ``x`` over its last dimension; with ``residual`` of ``s = residual + dropout(x, p)``, and then
    ``(y, s)`` is returned, s the stream for the next residual.

    ``weight`` and ``bias`` are ``(features,)``; fp32 ones beside 16-bit activations are read, and their gradients written,
    in fp32.  ``p``, ``seed`` and ``site`` as :func:`counter_dropout` has them (``p`` > 0 needs ``residual``).  The result has
    the compute dtype of ``x`` and ``residual`` (the loss's rule).  Gradients for every tensor, through y and s; once
    differentiable.  A training call keeps s (x without ``residual``, both with fp32 parameters beside 16-bit tensors) and two
    fp32 numbers a row.  ``backend`` as :func:`distillation_loss` has it."""
    entry = "layer_norm"
    check_tensors(entry, "none", x, weight=weight, bias=bias, residual=residual)
    check_shape(entry, "weight", weight, (x.shape[-1],))
    check_shape(entry, "bias", bias, (x.shape[-1],))
    check_shape(entry, "residual", residual, x.shape)
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"{entry}: eps must be finite and >= 0, got {eps}")
    p, seed, seed_tensor = check_dropout(entry, p, seed, site, x.device)
    if p > 0.0 and residual is None:
        raise ValueError(f"{entry}: p > 0 needs residual; use counter_dropout in front of a norm without one")
    kernels = use_kernels(backend, x, entry)
    dtype = default_compute_dtype(x, residual)
    if not kernels or x.numel() == 0:
        return _torch(x, weight, bias, residual, eps, p, seed, seed_tensor, site, dtype)
    x2 = x if x.ndim == 2 else x.reshape(-1, x.shape[-1])
    r2 = residual if residual is None or x.ndim == 2 else residual.reshape(-1, x.shape[-1])
    got = _native.torch_ops().layer_norm(x2, weight, bias, r2, eps, p, seed, site, seed_tensor, dtype,
                                         needs_function(x, weight, bias, residual))
    got = got if x.ndim == 2 else [t.reshape(x.shape) for t in got]
    return got[0] if residual is None else (got[0], got[1])
