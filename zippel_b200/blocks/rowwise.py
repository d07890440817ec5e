"""Layer norm, dropout and their join by a residual sum, on the B200 kernels.

    layer_norm(x, weight, bias, eps)                 what nn.LayerNorm computes over the last axis
    dropout(x, p, state)                             what nn.Dropout does in training
    dropout_add_layer_norm(x, residual, ...)         s = residual + dropout(x) and layer_norm(s), both
                                                     returned: the join of two layers of a residual network

fp32, fp16 and bf16, any leading axes, any width of the last; rows that lie one distance apart, a width at
least, are read where they are, others (expanded or overlapping ones) from a copy.  Sums and row statistics
are fp32, each result is rounded once, and sums over rows (the gradients of weight and bias) are taken in a
fixed order.  First order only, as every function of this package.  Calls under ``torch.jit.trace`` and
``make_fx`` are refused: they would leave a constant in the trace.

Dropout stores no mask: which elements are kept follows from ``state``, two int64 on the device (seed and
offset), and each element's number in the tensor, so the backward finds them again.  ``dropout_state``
draws one from torch's generator of the device, which makes a call repeatable by ``torch.manual_seed``
and under activation checkpointing, and gives every replay of a recorded CUDA graph its own.  One state
is one mask: calls that are to drop independently of each other need a state each.

``ResidualNorm`` is the join as a module, for ``rad_func`` of a block (``blocks.eso2.radial_mlp`` runs it,
``nn.LayerNorm`` by itself and ``nn.Dropout`` on these functions) or on its own.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from .. import _lib


def _native():
    """The extension module over ``libzippel_b200.so`` (``csrc/zp_rowwise_torch.cpp``): arguments are
    checked, laid out and recorded for autograd there."""
    global _module
    if _module is None:
        _lib.load()                            # (says what to do where nothing has been built)
        try:
            from .. import _rowwise as _module
        except ImportError as e:               # built without a torch, or for another one
            raise RuntimeError("the functions on tensors are missing or for another torch: build them with "
                               f"`python -m zippel_b200.build` ({e})") from e
    return _module


_module = None


def dropout_state(device) -> torch.Tensor:
    """(seed, offset) for one call, drawn from torch's generator of ``device``."""
    return torch.empty(2, dtype=torch.int64, device=device).random_()


def _threshold(p) -> int:
    """How many of 65536 are dropped."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"a probability is between 0 and 1: {p}")
    return math.floor(65536 * p + 0.5)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis.  ``weight`` and ``bias`` are of
    x's type or float32, and either may be missing."""
    return (_module or _native()).layer_norm(x, weight, bias, eps)


def dropout(x: torch.Tensor, p: float, state: torch.Tensor | None = None) -> torch.Tensor:
    """``x / keep`` where an element is kept and 0 where it is not, the latter with probability ``p``
    rounded to a multiple of 2^-16; keep is one minus that, so the mean is x.  ``x`` itself where
    that is 0 (no state is needed then)."""
    return (_module or _native()).dropout(x, p, state)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, p: float = 0.0,
                           state: torch.Tensor | None = None, eps: float = 1e-5):
    """``(y, s)``: ``s = residual + dropout(x, p, state)``, rounded to x's type, and
    ``y = layer_norm(s, weight, bias, eps)`` of s as it is returned, in one pass each way.  ``p = 0``
    (evaluation): no state is needed."""
    return (_module or _native()).dropout_add_layer_norm(x, residual, weight, bias, p, state, eps)


class ResidualNorm(nn.Module):
    """``layer_norm(x + dropout(layers(x)))``: some layers of one width with the residual around them
    and the norm behind.  ``layers`` are modules; within a block's ``rad_func`` they run on the library's
    kernels as the rest of it does."""

    def __init__(self, layers, width: int, p: float = 0.0, eps: float = 1e-5):
        super().__init__()
        _threshold(p)
        self.layers = layers if isinstance(layers, nn.Sequential) else nn.Sequential(*layers)
        self.p, self.eps = float(p), float(eps)
        self.weight = nn.Parameter(torch.ones(width))
        self.bias = nn.Parameter(torch.zeros(width))

    def join(self, x: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
        """The norm of x and what ``layers`` made of it."""
        p = self.p if self.training else 0.0
        state = dropout_state(h.device) if _threshold(p) else None
        weight, bias = (t if t.dtype == torch.float32 else t.to(h.dtype) for t in (self.weight, self.bias))
        return dropout_add_layer_norm(h, x, weight, bias, p, state, self.eps)[0]

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.join(x, self.layers(x))

    def extra_repr(self) -> str:
        return f"{self.weight.numel()}, p={self.p}, eps={self.eps}"
