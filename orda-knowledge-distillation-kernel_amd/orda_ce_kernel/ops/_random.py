"""Dropout's random bits: Philox4x32-10 of an element's index, the same in torch as in the kernels (csrc/philox.hpp), and
where a call's seed comes from."""
from __future__ import annotations

import math

import torch

__all__ = ["check_dropout", "kept_factors", "threshold_of"]

_MASK = 0xFFFFFFFF


def threshold_of(p: float) -> int:
    """p in steps of 2^-16, the nearest."""
    return math.floor(p * 65536.0 + 0.5)


def check_dropout(entry: str, p: float, seed, site: int, device: torch.device):
    """The checked (p, seed, seed's tensor or None)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{entry}: p must be in [0, 1], got {p}")
    if not isinstance(site, int) or not 0 <= site < 1 << 64:
        raise ValueError(f"{entry}: site must be an int in [0, 2^64), got {site!r}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise ValueError(f"{entry}: a seed tensor must be one int64 on {device}, got {seed.dtype} {tuple(seed.shape)} on "
                             f"{seed.device}")
        return p, 0, seed.reshape(1)
    if seed is None:
        if threshold_of(p) == 0:
            return p, 0, None
        if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{entry}: a captured call would repeat one seed with every replay; pass seed= as an int64 tensor "
                               "on the device and change it between replays")
        # (torch.manual_seed; no device work, whatever torch.device() or the default device says)
        return p, int(torch.randint(1 << 62, (), dtype=torch.int64, device="cpu")), None
    if isinstance(seed, bool) or not isinstance(seed, int) or not 0 <= seed < 1 << 64:
        raise ValueError(f"{entry}: seed must be an int in [0, 2^64) or an int64 tensor, got {seed!r}")
    return p, seed, None


def _times(x: torch.Tensor, m: int):
    """(high, low) 32 bits of x m, in int64."""
    y = x * m  # (wraps; its 64 bits are the product's)
    return (y >> 32) & _MASK, y & _MASK


def kept_factors(shape, p: float, seed: int, seed_tensor, site: int, device: torch.device) -> torch.Tensor:
    """0 where an element of a tensor of this shape is dropped, 1 / (1 - p) elsewhere, fp32."""
    n, drop = math.prod(shape), threshold_of(p)
    index = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    zero = torch.zeros_like(index)
    c = [index & _MASK, index >> 32, zero + (site & _MASK), zero + (site >> 32)]
    if seed_tensor is None:
        k = [zero[:1] + (seed & _MASK), zero[:1] + (seed >> 32)]
    else:
        k = [seed_tensor & _MASK, (seed_tensor >> 32) & _MASK]
    for _ in range(10):
        (h0, l0), (h1, l1) = _times(c[0], 0xD2511F53), _times(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k[0], l1, h0 ^ c[3] ^ k[1], l0]
        k = [(k[0] + 0x9E3779B9) & _MASK, (k[1] + 0xBB67AE85) & _MASK]
    words = torch.stack(c, 1)
    bits = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n].view(shape)
    return (bits >= drop).float() * (65536.0 / (65536 - drop) if drop < 65536 else 0.0)
