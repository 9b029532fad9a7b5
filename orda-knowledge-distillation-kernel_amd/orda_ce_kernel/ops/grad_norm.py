"""The norm over all gradients of a model, and their clipping: what follows the loss's backward pass.

    total = (sum |g|^p)^(1/p), p = 1, 2 or infinity        g *= min(1, max_norm / (total + 1e-6))

Two kernels over a table of tensors (one launch each per dtype and up to 320 tensors) and one that adds up the norm's partial sums;
sums are fp64 in a fixed order and the factor is formed on the device, so nothing synchronises the host.  The tables are
built in csrc/torch_ops.cpp.  No counterpart in the reference, whose training loop calls torch.
"""
from __future__ import annotations

import math

import torch

from .. import _native
from ._layers import use_kernels

__all__ = ["clip_grad_norm_", "grad_norm"]


def _listed(tensors) -> list:
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def _check_norm(entry: str, norm_type) -> float:
    norm_type = float(norm_type)
    if norm_type not in (1.0, 2.0, math.inf):
        raise ValueError(f"{entry}: norm_type must be 1, 2 or infinity, got {norm_type}")
    return norm_type


def _check_grad(entry: str, g: torch.Tensor, device) -> None:
    if g.layout is not torch.strided:
        raise ValueError(f"{entry}: gradients must be dense, got layout {g.layout}")
    if g.device != device:
        raise ValueError(f"{entry}: gradients must be on one device, got {device} and {g.device}")
    if g.dtype not in _native.DTYPE:
        raise ValueError(f"{entry}: gradients must be bfloat16, float16 or float32, got {g.dtype}")


def _norm_torch(grads, norm_type: float) -> torch.Tensor:
    return torch.linalg.vector_norm(
        torch.stack([torch.linalg.vector_norm(g.detach(), norm_type, dtype=torch.float64) for g in grads]), norm_type
    ).float()


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a is b or (a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()
                      and a.dtype == b.dtype and a.device == b.device)


def _clip_torch(entry, params, outs, max_norm, norm_type, error_if_nonfinite, total_norm):
    grads, dests, seen = [], [], {}
    for i, p in enumerate(params):
        g = p.grad
        if g is None:
            continue
        k = seen.setdefault(id(p), i)
        if k != i:
            if outs is not None and not _same_place(outs[k], outs[i]):
                raise ValueError(f"{entry}: parameters {k} and {i} are one, their out tensors are not")
            continue
        _check_grad(entry, g, grads[0].device if grads else g.device)
        if outs is not None:
            o = outs[i]
            if o.shape != g.shape or o.device != g.device or o.dtype not in _native.DTYPE:
                raise ValueError(f"{entry}: out[{i}] must be a bfloat16, float16 or float32 tensor of shape "
                                 f"{tuple(g.shape)} on {g.device}")
            dests.append(o)
        grads.append(g)
    if total_norm is None:
        total = _norm_torch(grads, norm_type)
    elif total_norm.numel() != 1 or total_norm.device != grads[0].device:
        raise ValueError(f"{entry}: total_norm must be a one-element tensor on {grads[0].device}")
    else:
        total = total_norm.detach().float().reshape(())
    if error_if_nonfinite and not bool(torch.isfinite(total)):
        raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it cannot "
                           "be clipped. To disable this error and scale the gradients by the non-finite norm anyway, set "
                           "`error_if_nonfinite=False`")
    factor = (max_norm / (total + 1e-6)).clamp(max=1.0)
    for g, o in zip(grads, dests or grads):
        o.copy_(g.float() * factor)
    return total


@torch._dynamo.disable
@torch.no_grad()
def grad_norm(tensors, norm_type: float = 2.0, *, backend: str = "auto") -> torch.Tensor:
    """The ``norm_type`` norm (1, 2 or infinity) over all elements of the tensors, a 0-dim fp32 tensor on their device.
    bf16, fp16 and fp32 tensors may be mixed.  No tensors: 0 (on the CPU).  For gradients sharded over ranks, reduce
    ``grad_norm(...) ** 2`` over the ranks and pass its root to :func:`clip_grad_norm_` as ``total_norm``."""
    norm_type = _check_norm("grad_norm", norm_type)
    grads = _listed(tensors)
    for g in grads:
        if not isinstance(g, torch.Tensor):
            raise TypeError(f"grad_norm: expected tensors, got {type(g).__name__}")
    if not grads:
        return torch.zeros(())
    if use_kernels(backend, grads[0], "grad_norm"):
        return _native.torch_ops().grad_norm(grads, norm_type)
    for g in grads:
        _check_grad("grad_norm", g, grads[0].device)
    return _norm_torch(grads, norm_type)


@torch._dynamo.disable
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, *,
                    total_norm: torch.Tensor | None = None, out=None, backend: str = "auto") -> torch.Tensor:
    """Scale the parameters' gradients by ``min(1, max_norm / (total + 1e-6))`` in place and return their total norm, as
    ``torch.nn.utils.clip_grad_norm_`` does, without synchronising the host (but for ``error_if_nonfinite``).

    Parameters without a gradient are left out; one that is listed twice counts once (and has one ``out`` tensor).
    ``total_norm`` (a one-element tensor): the norm to scale by, instead of these gradients' own.  ``out``: one tensor per
    parameter (any of the three dtypes, the gradient's shape) that receives the scaled gradient, which itself stays as it
    is: the fp32 buffers of a mixed-precision optimizer.  Tensors that are written must not share memory with any other of
    the call."""
    entry = "clip_grad_norm_"
    norm_type, max_norm = _check_norm(entry, norm_type), float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"{entry}: max_norm must be >= 0, got {max_norm}")
    params = _listed(parameters)
    outs = None if out is None else _listed(out)
    if outs is not None and len(outs) != len(params):
        raise ValueError(f"{entry}: out must have one tensor per parameter ({len(params)}), got {len(outs)}")
    if total_norm is not None and not isinstance(total_norm, torch.Tensor):
        raise ValueError(f"{entry}: total_norm must be a one-element tensor, got {type(total_norm).__name__}")
    first = next((p.grad for p in params if p.grad is not None), None)
    if first is None:
        return torch.zeros(()) if total_norm is None else total_norm
    if use_kernels(backend, first, entry):
        return _native.torch_ops().clip(params, max_norm, norm_type, bool(error_if_nonfinite), total_norm, outs)
    with torch.no_grad():
        return _clip_torch(entry, params, outs, max_norm, norm_type, error_if_nonfinite, total_norm)
