"""Dropout whose mask is never stored.

    y = residual + x keep / (1 - p)        dx = dy keep / (1 - p)

Whether an element is kept follows from 16 bits of Philox4x32-10 of its index, the seed and the site, which the backward
pass computes again (csrc/philox.hpp, csrc/rownorm.hip).  No counterpart in the reference.
"""
from __future__ import annotations

import torch

from .. import _native
from .._runtime import default_compute_dtype
from ._layers import check_shape, check_tensors, needs_function, use_kernels
from ._random import check_dropout, kept_factors

__all__ = ["counter_dropout"]


@torch._dynamo.disable
def counter_dropout(x: torch.Tensor, p: float, residual: torch.Tensor | None = None, *, seed: int | torch.Tensor | None = None,
                    site: int = 0, backend: str = "auto") -> torch.Tensor:
    """``residual + dropout(x, p)`` in one kernel, with its backward pass; no mask is stored.

    ``residual`` has ``x``'s shape.  ``p`` is taken to the nearest multiple of 2^-16, and kept elements are scaled by its
    ``1 / (1 - p)``; a dropped infinity or NaN leaves nothing.  Which elements are kept follows from ``seed``, ``site`` and
    the element's index in row-major order alone, so it does not depend on strides, dtype or device.  ``seed``: an int, an
    int64 tensor of one element on ``x``'s device (read by the kernels; what a captured graph needs, to be changed between
    replays), or None: drawn from torch's CPU generator.  ``site`` tells calls apart that share a seed.  The result has the
    compute dtype of ``x`` and ``residual``; once differentiable.  ``backend`` as :func:`distillation_loss` has it."""
    entry = "counter_dropout"
    check_tensors(entry, "none", x, residual=residual)
    check_shape(entry, "residual", residual, x.shape)
    p, seed, seed_tensor = check_dropout(entry, p, seed, site, x.device)
    kernels = use_kernels(backend, x, entry)
    dtype = default_compute_dtype(x, residual)
    if not kernels or x.numel() == 0:
        keep = kept_factors(x.shape, p, seed, seed_tensor, site, x.device)
        y = torch.where(keep > 0, x.to(dtype).float() * keep, 0.0)
        return (y if residual is None else y + residual.to(dtype).float()).to(dtype)
    return _native.torch_ops().dropout(x, residual, p, seed, site, seed_tensor, dtype, needs_function(x, residual))
