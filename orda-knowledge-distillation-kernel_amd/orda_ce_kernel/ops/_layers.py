"""What the projection and the feed-forward block share: argument checks, the compute dtype, operands as the kernels
read them."""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from .. import _native
from .._runtime import HAS_NATIVE, native_error

__all__ = ["ACTIVATIONS", "activation_torch", "check_tensors", "needs_function", "operand", "same_pitch", "use_kernels",
           "new_grad", "trim"]

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
    on_device = x.device.type == "cuda"
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
    """Whether autograd has to see the call: a gradient is wanted, or a forward-mode level is open (the Functions have no
    jvp, and autograd then refuses the call instead of dropping a tangent)."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def operand(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A 2-D operand as the kernels read it: rows in memory order, 16-byte aligned and zero-padded to 16 bytes.  Row-strided
    tensors that already are so stay where they are."""
    if t.dtype != dtype:
        t = t.to(dtype)
    mult = 4 if dtype == torch.float32 else 8
    rows, cols = t.shape
    if cols % mult:
        return F.pad(t, (0, -cols % mult))
    if t.stride(1) != 1 or (rows > 1 and (t.stride(0) % mult or t.stride(0) < cols)):
        t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def pitch(t: torch.Tensor) -> int:
    """Elements between the rows of an operand (one row: its length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def same_pitch(a: torch.Tensor, b: torch.Tensor):
    """Both operands with the same row pitch."""
    if pitch(a) != pitch(b):
        a, b = a.contiguous(), b.contiguous()
    return a, b


def rows_of(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A 2-D tensor with contiguous rows in `dtype` (any row pitch, any alignment)."""
    if t.dtype != dtype:
        t = t.to(dtype)
    if t.stride(1) != 1 and t.shape[1] > 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def new_grad(rows: int, cols: int, dtype: torch.dtype, device) -> torch.Tensor:
    """A gradient's buffer, its rows padded to 16 bytes."""
    mult = 4 if dtype == torch.float32 else 8
    return torch.empty((rows, cols + (-cols) % mult), dtype=dtype, device=device)


def trim(grad: torch.Tensor | None, cols: int, shape, dtype: torch.dtype):
    """The gradient in its tensor's shape and dtype, without the padding."""
    if grad is None:
        return None
    if grad.shape[1] != cols:
        grad = grad[:, :cols]
    if grad.dtype != dtype:
        grad = grad.to(dtype)
    return grad if grad.shape == shape else grad.reshape(shape)
