"""The token embedding.

    y[n] = scale W[t_n]        dW[v] = scale sum of dy[n] over t_n = v

One kernel copies the rows.  The gradient sorts the tokens (in LDS, while other workgroups fill dW with zeros) and adds up
each token's rows of dy in fp32 in the order of the batch, long runs of one token in parts that are joined afterwards: no
atomics, the same bits in every run (csrc/embed.hip).  No counterpart in the reference, whose models use torch.
"""
from __future__ import annotations

import math

import torch

from .. import _native
from .._runtime import default_compute_dtype
from ._layers import check_tensors, needs_function, use_kernels

__all__ = ["token_embedding"]


def _torch(ids, weight, scale, padding_idx, dtype):
    flat = ids.reshape(-1).long()
    known = (flat >= 0) & (flat < weight.shape[0])
    rows = weight[flat.where(known, 0)] if flat.numel() else weight.new_zeros((0, weight.shape[1])) + weight[:0].sum()
    if padding_idx is not None:
        rows = torch.where((flat == padding_idx)[:, None], rows.detach(), rows)
    return torch.where(known[:, None], rows.float() * scale, 0.0).to(dtype)


@torch._dynamo.disable
def token_embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None,
                    backend: str = "auto") -> torch.Tensor:
    """``scale * weight[ids]``, with its backward pass.

    ``ids`` is an int32 or int64 tensor of any shape, ``weight`` ``(vocab, hidden)``; the result is ``(*ids.shape, hidden)``
    in the compute dtype of ``weight`` (an active autocast dtype, else its own).  An id outside ``[0, vocab)``, such as -100
    behind a sequence, gives zeros and takes no part in the gradient; ``padding_idx`` is looked up and gets no gradient.
    The gradient is dense, in the weight's dtype, rounded once; once differentiable.  ``backend`` as
    :func:`distillation_loss` has it."""
    entry = "token_embedding"
    check_tensors(entry, "none", weight)
    if weight.ndim != 2 or weight.shape[0] == 0:
        raise ValueError(f"{entry}: weight must have shape (vocab, hidden), got {tuple(weight.shape)}")
    if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{entry}: ids must be an int32 or int64 tensor, got {getattr(ids, 'dtype', type(ids).__name__)}")
    if ids.device != weight.device:
        raise ValueError(f"{entry}: ids are on {ids.device}, weight on {weight.device}")
    scale = float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"{entry}: scale must be finite, got {scale}")
    if padding_idx is not None and not 0 <= padding_idx < weight.shape[0]:
        raise ValueError(f"{entry}: padding_idx must be in [0, {weight.shape[0]}), got {padding_idx}")
    kernels = use_kernels(backend, weight, entry)
    dtype = default_compute_dtype(weight)
    shape = (*ids.shape, weight.shape[1])
    if not kernels or ids.numel() == 0:
        return _torch(ids, weight, scale, padding_idx, dtype).reshape(shape)
    y = _native.torch_ops().embedding(ids.reshape(-1), weight, scale, -1 if padding_idx is None else int(padding_idx), dtype,
                                      needs_function(weight))
    return y.reshape(shape)
