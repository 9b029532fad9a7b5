"""Masked self-attention.

    z = scale q.k;  cap tanh(z / cap);  less slope_h |i - j|;      P = softmax over the keys that a query sees;      o = P v
    dv = P^T do      dz = P (do v^T - sum(do o))      dq = scale dz k      dk = scale dz^T q

One kernel forward, two backward, on the matrix cores, with the softmax in one pass over the keys; scores never reach
memory, and tiles that no query sees are not read (csrc/attn.hpp).  No counterpart in the reference, whose models use torch.
"""
from __future__ import annotations

import math

import torch

from .. import _native
from .._runtime import default_compute_dtype
from ._layers import check_shape, check_tensors, needs_function, use_kernels

__all__ = ["masked_attention"]


def _seen(B, S, causal, documents, prefix, device):
    """(B, S, S): whether query i sees key j."""
    at = torch.arange(S, device=device)
    seen = torch.ones(B, S, S, dtype=torch.bool, device=device)
    if causal:
        seen = (at[:, None] >= at[None]).expand(B, S, S)
        if prefix is not None:
            seen = seen | (at[None, None] < prefix[:, None, None])
    if documents is not None:
        seen = seen & (documents[:, :, None] == documents[:, None]) & (documents >= 0)[:, :, None]
    return seen


def _torch(q, k, v, causal, scale, softcap, slopes, documents, prefix, dtype):
    B, S, H, D = q.shape
    G = H // k.shape[2]
    seen = _seen(B, S, causal, documents, prefix, q.device)[:, None]
    if documents is not None:  # (padding rows may hold anything)
        real = (documents >= 0)[:, :, None, None]
        q, k, v = (torch.where(real, t, torch.zeros((), dtype=t.dtype, device=t.device)) for t in (q, k, v))
    qf = q.to(dtype).float().transpose(1, 2)
    kf, vf = (t.to(dtype).float().transpose(1, 2).repeat_interleave(G, 1) for t in (k, v))
    z = torch.matmul(qf, kf.transpose(2, 3).contiguous()) * scale
    if softcap:
        z = softcap * torch.tanh(z / softcap)
    if slopes is not None:
        at = torch.arange(S, device=q.device)
        z = z - slopes.view(1, H, 1, 1) * (at[:, None] - at[None]).abs()
    some = seen.any(-1, keepdim=True)
    z = torch.where(seen, z, -math.inf)
    p = torch.softmax(torch.where(some, z, 0.0), -1)
    o = torch.matmul(torch.where(some, p, 0.0), vf).transpose(1, 2).to(dtype)
    # (the gradient from above of a padding row may hold anything too)
    return o if documents is None else torch.where(real, o, torch.zeros((), dtype=dtype, device=o.device))


def _integers(entry, name, t, shape, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{entry}: {name} must be an int32 or int64 tensor, got {getattr(t, 'dtype', type(t).__name__)}")
    check_shape(entry, name, t, shape)
    if t.device != device:
        raise ValueError(f"{entry}: {name} is on {t.device}, q on {device}")
    return t.clamp(-1, 2**31 - 1).to(torch.int32).contiguous() if t.dtype == torch.int64 else t.contiguous()


@torch._dynamo.disable
def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True, scale: float | None = None,
                     softcap: float = 0.0, slopes: torch.Tensor | None = None, documents: torch.Tensor | None = None,
                     prefix: torch.Tensor | None = None, backend: str = "auto") -> torch.Tensor:
    """Self-attention over whole sequences, with its backward pass.

    ``q`` is ``(batch, length, heads, head_dim)``, ``k`` and ``v`` ``(batch, length, kv_heads, head_dim)`` with ``heads`` a
    multiple of ``kv_heads`` (query head h reads head ``h // (heads // kv_heads)``); slices of one projection's output serve
    as they are.  The result is ``(batch, length, heads, head_dim)``.  ``scale`` (default ``head_dim ** -0.5``) multiplies the
    products; ``softcap`` > 0 caps them to ``softcap * tanh(z / softcap)``, at any cap with the precision of the score;
    ``slopes`` (``(heads,)``) takes ``slopes[h] * |i - j|`` off.  ``causal``: query i sees the keys up to i, and with ``prefix`` (``(batch,)``) also those below
    ``prefix[b]`` (without ``causal`` it sees them all).  ``documents`` (``(batch, length)``): only keys with the query's own
    number (int64 numbers past 2^31 - 1 count as that one); a negative number is padding, which sees nothing and is not
    seen, whatever it holds: zeros come out, and zero gradients.

    On the kernels bf16 and fp16 with head_dim up to 128 (multiples of 8 are read in place, others are copied) and batches
    up to 65535.  The compute dtype is the loss's rule; fp32 tensors run on ``backend="torch"`` or under autocast.  Scores and
    sums are fp32 (a score's size times 2^-24 is what its probability may be off in the backward pass).  Probabilities and
    their gradients are rounded to the compute dtype as operands of products, in fp16 lifted so that small ones keep its 11
    bits; the gradients in two parts up to a length of 64, beyond in one (documents of any length in longer rows too), which
    leaves the gradients of q and k off by 2.4e-3 of their norm in bf16 instead of the 1.7e-3 of their own rounding, and by
    3e-4 instead of 2e-4 in fp16.  A training call keeps q, k, v, the result, what its rounding left (a second tensor of its
    size) and an fp32 number a query and head.
    A value that is not finite, in a row that a query does not see, may still reach it where a query of the same 128 (from
    the sequence's start) sees a row of the value's 64 (padding excepted).  Once differentiable, in q, k and v.
    ``backend`` as :func:`distillation_loss` has it."""
    entry = "masked_attention"
    check_tensors(entry, "none", q, k=k, v=v, slopes=slopes)
    if q.ndim != 4:
        raise ValueError(f"{entry}: q must have shape (batch, length, heads, head_dim), got {tuple(q.shape)}")
    B, S, H, D = q.shape
    if k.ndim != 4 or k.shape[2] == 0 or H % k.shape[2] != 0:
        raise ValueError(f"{entry}: k must have shape ({B}, {S}, kv_heads, {D}) with kv_heads a divisor of {H}, got {tuple(k.shape)}")
    check_shape(entry, "k", k, (B, S, k.shape[2], D))
    check_shape(entry, "v", v, k.shape)
    check_shape(entry, "slopes", slopes, (H,))
    if slopes is not None and slopes.requires_grad:
        raise ValueError(f"{entry}: slopes are constants; they have no gradient")
    documents = _integers(entry, "documents", documents, (B, S), q.device)
    prefix = _integers(entry, "prefix", prefix, (B,), q.device)
    scale = D ** -0.5 if scale is None else float(scale)
    softcap = float(softcap)
    if not abs(scale) <= 1e38:
        raise ValueError(f"{entry}: scale must be finite in fp32, up to 1e38, got {scale}")
    if not (softcap >= 0.0 and math.isfinite(softcap)):
        raise ValueError(f"{entry}: softcap must be finite and >= 0, got {softcap}")
    if softcap:  # (a cap below the one leaves scores of 0 and one past the other the scores as they are, in fp32)
        softcap = min(max(softcap, 1e-24), 1e30)
    kernels = use_kernels(backend, q, entry)
    dtype = default_compute_dtype(q, k, v)
    slopes = None if slopes is None else slopes.detach().float().contiguous()
    if not kernels or q.numel() == 0:
        return _torch(q, k, v, causal, scale, softcap, slopes, documents, prefix, dtype)
    if dtype == torch.float32:
        raise ValueError(f"{entry}: the kernels take bfloat16 and float16; cast, use autocast, or pass backend='torch'")
    if D > 128:
        raise ValueError(f"{entry}: the kernels take head_dim up to 128, got {D}; pass backend='torch'")
    return _native.torch_ops().attention(q, k, v, slopes, documents, prefix, bool(causal), scale, softcap, dtype,
                                         needs_function(q, k, v))
