"""Layer norm, dropout and their join by a residual sum, on the B200 kernels.

    layer_norm(x, weight, bias, eps)                 what nn.LayerNorm computes over the last axis
    dropout(x, p, state)                             what nn.Dropout does in training
    dropout_add_layer_norm(x, residual, ...)         s = residual + dropout(x) and layer_norm(s), both
                                                     returned: the join of two layers of a residual network

fp32, fp16 and bf16, any leading axes, any width of the last; rows of a wider array are read where they
lie.  Sums and row statistics are fp32, each result is rounded once, and sums over rows (the gradients
of weight and bias) are taken in a fixed order.  First order only, as every function of this package.

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
from torch.autograd import forward_ad

from .. import _lib

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def dropout_state(device) -> torch.Tensor:
    """(seed, offset) for one call, drawn from torch's generator of ``device``."""
    return torch.empty(2, dtype=torch.int64, device=device).random_()


def _need(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{what} needs CUDA tensors: there is no CPU path")
    if x.dtype not in _TYPES:
        raise TypeError(f"{what} takes float32, float16 and bfloat16, not {x.dtype}")


def _need_alike(x, other, what: str, shape=None) -> None:
    """``other`` is of x's type and shape (or of ``shape``) and on its device."""
    shape = x.shape if shape is None else shape
    if other.shape != shape:
        raise ValueError(f"{what} has shape {tuple(other.shape)}, expected {tuple(shape)}")
    if other.device != x.device:
        raise RuntimeError(f"{what} is on {other.device}, x on {x.device}")
    if other.dtype != x.dtype:
        raise TypeError(f"{what} is {other.dtype}, x is {x.dtype}")


def _need_params(x, weight, bias) -> None:
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"a layer norm over the last axis of a tensor of shape {tuple(x.shape)}")
    for t, what in ((weight, "the weight"), (bias, "the bias")):
        if t is None:
            continue
        if t.shape != x.shape[-1:]:
            raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(x.shape[-1:])}")
        if t.device != x.device:
            raise RuntimeError(f"{what} is on {t.device}, x on {x.device}")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError(f"{what} is {t.dtype}; with x in {x.dtype} it may be that or float32")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"the weight is {weight.dtype}, the bias {bias.dtype}")


def _threshold(p) -> int:
    """How many of 65536 are dropped."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"a probability is between 0 and 1: {p}")
    return math.floor(65536 * p + 0.5)


def _need_state(x, state) -> None:
    if state is None:
        raise ValueError("dropout with p > 0 needs a state: dropout_state(device) draws one")
    if state.dtype != torch.int64 or state.numel() != 2 or not state.is_contiguous():
        raise ValueError("a dropout state is two int64 one behind the other (seed, offset)")
    if state.device != x.device:
        raise RuntimeError(f"the dropout state is on {state.device}, x on {x.device}")


def _recorded(*tensors) -> bool:
    """Whether autograd has to see the call: for a gradient, or to refuse tangents (forward mode)."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _rows(x: torch.Tensor):
    """``x`` or a copy that the kernels can read, its rows, width and the elements between two rows."""
    w = x.shape[-1] if x.dim() else 1
    if x.is_contiguous():
        return x, x.numel() // w if w else 0, w, w
    if x.dim() == 2:
        r, (ld, step) = x.shape[0], x.stride()
        if (step == 1 or w == 1) and ld >= w:
            return x, r, w, ld
    elif x.stride(-1) == 1 and x.numel():
        try:                                   # leading axes that are one row behind the other
            v = x.view(-1, w)
        except RuntimeError:
            pass
        else:
            if v.stride(0) >= w or v.shape[0] == 1:
                return v, v.shape[0], w, max(v.stride(0), w)
    x = x.contiguous()
    return x, x.numel() // w if w else 0, w, w


def _ptr(t):
    return None if t is None else t.data_ptr()


def _new(x: torch.Tensor) -> torch.Tensor:
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _param_type(x, weight, bias) -> int:
    for t in (weight, bias):
        if t is not None:
            return _TYPES[t.dtype]
    return _TYPES[x.dtype]


def _work(x, rows, width):
    nbytes = _lib.load().zp_rowwise_work_bytes(rows, width)
    return torch.empty(nbytes, dtype=torch.uint8, device=x.device), nbytes


# ---- dropout -----------------------------------------------------------------------------------


def _dropped(x, p, state) -> torch.Tensor:
    y = _new(x)
    if y.numel():
        x, rows, width, ld = _rows(x)
        _lib.run(x.device, "zp_dropout", rows, width, _TYPES[x.dtype], x.data_ptr(), ld, p,
                 state.data_ptr(), y.data_ptr(), width)
    return y


class DropoutFunction(torch.autograd.Function):
    """``dropout`` with its gradient: the same call on the gradient of the result."""

    @staticmethod
    def forward(ctx, x, p: float, state):
        ctx.p = p
        ctx.save_for_backward(state)
        return _dropped(x.detach(), p, state)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        return _dropped(grad_y, ctx.p, *ctx.saved_tensors), None, None


def dropout(x: torch.Tensor, p: float, state: torch.Tensor | None = None) -> torch.Tensor:
    """``x / keep`` where an element is kept and 0 where it is not, the latter with probability ``p``
    rounded to a multiple of 2^-16; keep is one minus that, so the mean is x.  ``x`` itself where
    that is 0 (no state is needed then)."""
    _need(x, "dropout")
    if _threshold(p) == 0:
        return x
    _need_state(x, state)
    if _recorded(x):
        return DropoutFunction.apply(x, float(p), state)
    return _dropped(x, p, state)


# ---- layer norm --------------------------------------------------------------------------------


def _norm(x, weight, bias, eps: float, keep: bool):
    """y, and with ``keep`` the rows' mean and 1/std one behind the other."""
    y = _new(x)
    x, rows, width, ld = _rows(x)
    stats = torch.empty(2, rows, dtype=torch.float32, device=x.device) if keep else None
    at = stats.data_ptr() if keep else None
    _lib.run(x.device, "zp_layernorm_forward", rows, width, _TYPES[x.dtype], x.data_ptr(), ld,
             _param_type(x, weight, bias), _ptr(weight), _ptr(bias), eps, y.data_ptr(), at,
             at + 4 * rows if keep else None)
    return y, x, stats


def _param_grads(weight, bias, want_w: bool, want_b: bool):
    return (torch.empty_like(weight) if want_w else None, torch.empty_like(bias) if want_b else None)


class LayerNormFunction(torch.autograd.Function):
    """``layer_norm`` with its gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps: float):
        weight, bias = (None if t is None else t.detach().contiguous() for t in (weight, bias))
        y, x, stats = _norm(x.detach(), weight, bias, eps, True)
        ctx.shape = y.shape
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y):
        x, weight, bias, stats = ctx.saved_tensors
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        x, rows, width, ld = _rows(x)
        dy, _, _, ldy = _rows(grad_y)
        dx = torch.empty(ctx.shape, dtype=x.dtype, device=x.device) if want_x else None
        dw, db = _param_grads(weight, bias, want_w, want_b)
        work, nbytes = _work(x, rows, width) if want_w or want_b else (None, 0)
        _lib.run(x.device, "zp_layernorm_backward", rows, width, _TYPES[x.dtype], x.data_ptr(), ld,
                 _param_type(x, weight, bias), _ptr(weight), stats.data_ptr(), stats.data_ptr() + 4 * rows,
                 dy.data_ptr(), ldy, _ptr(dx), _ptr(dw), _ptr(db), _ptr(work), nbytes)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis.  ``weight`` and ``bias`` are of
    x's type or float32, and either may be missing."""
    _need(x, "layer_norm")
    _need_params(x, weight, bias)
    if _recorded(x, weight, bias):
        return LayerNormFunction.apply(x, weight, bias, float(eps))
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    return _norm(x, weight, bias, eps, False)[0]


# ---- the join ----------------------------------------------------------------------------------


def _add_norm(x, residual, weight, bias, p: float, state, eps: float, keep: bool):
    y, s = _new(x), _new(x)
    x, rows, width, ld = _rows(x)
    residual, _, _, ldr = _rows(residual)
    stats = torch.empty(2, rows, dtype=torch.float32, device=x.device) if keep else None
    at = stats.data_ptr() if keep else None
    _lib.run(x.device, "zp_add_layernorm_forward", rows, width, _TYPES[x.dtype], x.data_ptr(), ld,
             residual.data_ptr(), ldr, p, _ptr(state), _param_type(x, weight, bias), _ptr(weight),
             _ptr(bias), eps, s.data_ptr(), y.data_ptr(), at, at + 4 * rows if keep else None)
    return y, s, stats


class DropoutAddLayerNormFunction(torch.autograd.Function):
    """``dropout_add_layer_norm`` with its gradients; ``state`` None: nothing is dropped."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, p: float, state, eps: float):
        weight, bias = (None if t is None else t.detach().contiguous() for t in (weight, bias))
        y, s, stats = _add_norm(x.detach(), residual.detach(), weight, bias, p, state, eps, True)
        ctx.p = p
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(s, weight, bias, stats, state)
        return y, s

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_y, grad_s):
        s, weight, bias, stats, state = ctx.saved_tensors
        want_x, want_res, want_w, want_b = ctx.needs_input_grad[:4]
        if grad_y is None and grad_s is None:
            return (None,) * 7
        _, rows, width, _ = _rows(s)
        dy, ldy = (None, 0) if grad_y is None else _rows(grad_y)[::3]
        ds, lds = (None, 0) if grad_s is None else _rows(grad_s)[::3]
        # without dropout the two gradients are one, and one tensor
        dres = _new(s) if want_res or want_x and state is None else None
        dx = _new(s) if want_x and state is not None else None
        dw, db = _param_grads(weight, bias, want_w, want_b)
        work, nbytes = _work(s, rows, width) if want_w or want_b else (None, 0)
        _lib.run(s.device, "zp_add_layernorm_backward", rows, width, _TYPES[s.dtype], s.data_ptr(),
                 _param_type(s, weight, bias), _ptr(weight), stats.data_ptr(), stats.data_ptr() + 4 * rows,
                 _ptr(dy), ldy, _ptr(ds), lds, ctx.p, _ptr(state), _ptr(dx), _ptr(dres), _ptr(dw),
                 _ptr(db), _ptr(work), nbytes)
        return dres if state is None and want_x else dx, dres if want_res else None, dw, db, None, None, None


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, p: float = 0.0,
                           state: torch.Tensor | None = None, eps: float = 1e-5):
    """``(y, s)``: ``s = residual + dropout(x, p, state)``, rounded to x's type, and
    ``y = layer_norm(s, weight, bias, eps)`` of s as it is returned, in one pass each way.  ``p = 0``
    (evaluation): no state is needed."""
    _need(x, "dropout_add_layer_norm")
    _need_params(x, weight, bias)
    _need_alike(x, residual, "the residual")
    if _threshold(p) == 0:
        p, state = 0.0, None
    else:
        _need_state(x, state)
    if _recorded(x, residual, weight, bias):
        return DropoutAddLayerNormFunction.apply(x, residual, weight, bias, float(p), state, float(eps))
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    return _add_norm(x, residual, weight, bias, p, state, eps, False)[:2]


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
