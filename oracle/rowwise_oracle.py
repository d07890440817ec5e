"""Layer norm, dropout and their residual join in FP64 on the CPU, from their definitions (a reference
for the kernels, never shipped code).  The generator is Philox-4x32-10 (Salmon, Moraes, Dror, Shaw,
"Parallel random numbers: as easy as 1, 2, 3", SC 2011) in Python's integers."""

from __future__ import annotations

import math

import torch


def philox(counter, key) -> list[int]:
    """Four 32-bit words of a counter (four words) under a key (two)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(n: int, p: float, state, first: int = 0) -> torch.Tensor:
    """Which of elements first .. first + n - 1 are kept."""
    t = math.floor(65536 * p + 0.5)
    seed, offset = (int(v) % 2 ** 64 for v in state)
    split = lambda v: (v & 0xFFFFFFFF, v >> 32)                                    # noqa: E731
    halves = []
    for g in range(first // 8, (first + n + 7) // 8):
        halves += [h for w in philox((*split(g), *split(offset)), split(seed)) for h in (w & 0xFFFF, w >> 16)]
    return torch.tensor(halves[first % 8:first % 8 + n]) >= t


def factors(shape, p: float, state) -> torch.Tensor:
    t = math.floor(65536 * p + 0.5)
    keep = kept(math.prod(shape), p, state).view(shape).double()
    return keep * (65536 / (65536 - t) if t < 65536 else 0.0)


def layer_norm(x, weight, bias, eps: float):
    """y, z (normalised rows) and rstd."""
    xc = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    y = xc * rstd
    y = y if weight is None else y * weight
    return (y if bias is None else y + bias), xc * rstd, rstd


def layer_norm_vjp(z, rstd, weight, gy):
    """Gradients of the rows, the weight and the bias."""
    gz = gy if weight is None else gy * weight
    gx = rstd * (gz - gz.mean(-1, keepdim=True) - z * (gz * z).mean(-1, keepdim=True))
    lead = tuple(range(gy.dim() - 1))
    return gx, (gy * z).sum(lead), gy.sum(lead)
