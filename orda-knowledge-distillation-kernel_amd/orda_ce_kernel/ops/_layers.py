"""What the projection and the feed-forward block share: argument checks, the choice between the kernels and torch, and when
autograd has to see a call."""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from .. import _native
from .._runtime import HAS_NATIVE, native_error

__all__ = ["ACTIVATIONS", "activation_torch", "check_shape", "check_tensors", "needs_function", "use_kernels"]

ACTIVATIONS = tuple(_native.ACTIVATION)


def activation_torch(name: str, x: torch.Tensor) -> torch.Tensor:
    if name == "none":
        return x
    if name == "gelu_tanh":
        return F.gelu(x, approximate="tanh")
    return {"relu": F.relu, "gelu": F.gelu, "silu": F.silu, "sigmoid": torch.sigmoid}[name](x)


def use_kernels(backend: str, x: torch.Tensor, entry: str) -> bool:
    """Whether the call runs on the HIP kernels (the loss's rule: never a silent fallback on a HIP device)."""
    if backend not in ("auto", "triton", "hip", "torch"):
        raise ValueError(f"backend must be 'auto', 'triton', 'hip', or 'torch', got {backend!r}")
    on_device = x.is_cuda
    if backend == "torch" or (backend == "auto" and not on_device):
        return False
    if not (HAS_NATIVE and on_device):
        raise RuntimeError(
            f"{entry}: backend={backend!r} on {x.device} tensors requires the HIP extension liborda_ce.so "
            f"({native_error() or 'loaded'}); pass backend='torch' to run the unfused PyTorch formulation"
        )
    return True


def check_tensors(entry: str, activation: str, x: torch.Tensor, **others) -> None:
    if activation not in _native.ACTIVATION:
        raise ValueError(f"{entry}: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if not isinstance(x, torch.Tensor) or x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"{entry}: x must be a tensor of shape (..., features), features > 0, got {getattr(x, 'shape', None)}")
    dev = x.device
    for name, t in (("x", x), *others.items()):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{entry}: {name} must be a tensor, got {type(t).__name__}")
        if t.device != dev:
            raise ValueError(f"{entry}: {name} is on {t.device}, x on {dev}")
        if t.dtype not in _native.DTYPE:
            raise ValueError(f"{entry}: {name} must be bfloat16, float16 or float32, got {t.dtype}")


def check_shape(entry: str, name: str, t: torch.Tensor | None, shape: tuple) -> None:
    if t is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{entry}: {name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def needs_function(*tensors) -> bool:
    """Whether autograd has to see the call: a gradient is wanted, or a forward-mode level is open (the nodes have no jvp,
    and autograd then refuses the call instead of dropping a tangent)."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
