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


def _type(x: torch.Tensor, what: str) -> int:
    """The library's number of x's type, if it runs on x at all."""
    if not x.is_cuda:
        raise RuntimeError(f"{what} needs CUDA tensors: there is no CPU path")
    code = _TYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"{what} takes float32, float16 and bfloat16, not {x.dtype}")
    return code


def _param_type(x, weight, bias, code: int) -> int:
    """The type of weight and bias, which are checked against x (of type ``code``)."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"a layer norm over the last axis of a tensor of shape {tuple(x.shape)}")
    size, found = x.shape[-1:], None
    for t in (weight, bias):
        if t is None:
            continue
        if t.shape != size:
            raise ValueError(f"weight or bias has shape {tuple(t.shape)}, expected {tuple(size)}")
        if t.get_device() != x.get_device():
            raise RuntimeError(f"weight or bias is on {t.device}, x on {x.device}")
        if t.dtype != x.dtype and t.dtype != torch.float32:
            raise TypeError(f"weight or bias is {t.dtype}; with x in {x.dtype} it may be that or float32")
        if found is not None and t.dtype != found:
            raise TypeError(f"the weight is {found}, the bias {t.dtype}")
        found = t.dtype
    return code if found is None else _TYPES[found]


def _threshold(p) -> int:
    """How many of 65536 are dropped."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"a probability is between 0 and 1: {p}")
    return math.floor(65536 * p + 0.5)


def _need_state(x, state) -> None:
    if state is None:
        raise ValueError("dropout with p > 0 needs a state: dropout_state(device) draws one")
    if state.dtype != torch.int64 or state.shape != (2,) or not state.is_contiguous():
        raise ValueError("a dropout state is two int64 one behind the other (seed, offset)")
    if state.get_device() != x.get_device():
        raise RuntimeError(f"the dropout state is on {state.device}, x on {x.device}")


def _recorded(*tensors) -> bool:
    """Whether autograd has to see the call: for a gradient, or to refuse tangents (forward mode)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return forward_ad._current_level >= 0


def _rows(x: torch.Tensor):
    """``x`` or a copy that the kernels can read, its rows, width and the elements between two rows."""
    shape = x.shape
    w = shape[-1] if shape else 1
    if x.is_contiguous():
        return x, x.numel() // w if w else 0, w, w
    if len(shape) == 2:
        ld, step = x.stride()
        if (step == 1 or w == 1) and ld >= w:
            return x, shape[0], w, ld
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
    """Like x, row behind row."""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _stats(x, rows: int):
    """Room for the rows' mean and 1/std one behind the other, and both addresses."""
    stats = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    at = stats.data_ptr()
    return stats, at, at + 4 * rows


def _param_grads(weight, bias, want_w: bool, want_b: bool, rows: int):
    """Room for the gradients that are wanted, and for their sums."""
    if not (want_w or want_b):
        return None, None, None, 0
    dw = torch.empty_like(weight) if want_w else None
    db = torch.empty_like(bias) if want_b else None
    t = dw if want_w else db
    nbytes = _lib.load().zp_rowwise_work_bytes(rows, t.shape[0])
    return dw, db, torch.empty(nbytes, dtype=torch.uint8, device=t.device), nbytes


def _first_order(backward):
    """``once_differentiable`` where a graph of the backward is asked for; its bookkeeping, a tenth of
    a small call, is spared where none is."""
    once = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return (once if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


# ---- dropout -----------------------------------------------------------------------------------


def _dropped(x, p: float, state) -> torch.Tensor:
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
        return _dropped(x, p, state)

    @staticmethod
    @_first_order
    def backward(ctx, grad_y):
        return _dropped(grad_y, ctx.p, *ctx.saved_tensors), None, None


def dropout(x: torch.Tensor, p: float, state: torch.Tensor | None = None) -> torch.Tensor:
    """``x / keep`` where an element is kept and 0 where it is not, the latter with probability ``p``
    rounded to a multiple of 2^-16; keep is one minus that, so the mean is x.  ``x`` itself where
    that is 0 (no state is needed then)."""
    _type(x, "dropout")
    if _threshold(p) == 0:
        return x
    _need_state(x, state)
    if _recorded(x):
        return DropoutFunction.apply(x, float(p), state)
    return _dropped(x, float(p), state)


# ---- layer norm --------------------------------------------------------------------------------


def _norm(x, weight, bias, eps: float, types, keep: bool):
    """y, x as it was read, and with ``keep`` the rows' mean and 1/std."""
    y = _new(x)
    x, rows, width, ld = _rows(x)
    stats, mean, rstd = _stats(x, rows) if keep else (None, None, None)
    _lib.run(x.device, "zp_layernorm_forward", rows, width, types[0], x.data_ptr(), ld, types[1], _ptr(weight),
             _ptr(bias), eps, y.data_ptr(), mean, rstd)
    return y, x, stats


class LayerNormFunction(torch.autograd.Function):
    """``layer_norm`` with its gradients; ``types``: the library's numbers of the rows' and the
    parameters' type."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps: float, types):
        weight, bias = _lined_up(weight), _lined_up(bias)
        y, read, stats = _norm(x, weight, bias, eps, types, True)
        ctx.types, ctx.shape = types, x.shape
        ctx.save_for_backward(read, weight, bias, stats)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, grad_y):
        x, weight, bias, stats = ctx.saved_tensors
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        x, rows, width, ld = _rows(x)
        dy, _, _, ldy = _rows(grad_y)
        dx = torch.empty(ctx.shape, dtype=x.dtype, device=x.device) if want_x else None
        dw, db, work, nbytes = _param_grads(weight, bias, want_w, want_b, rows)
        at = stats.data_ptr()
        _lib.run(x.device, "zp_layernorm_backward", rows, width, ctx.types[0], x.data_ptr(), ld, ctx.types[1],
                 _ptr(weight), at, at + 4 * rows, dy.data_ptr(), ldy, _ptr(dx), _ptr(dw), _ptr(db), _ptr(work), nbytes)
        return dx, dw, db, None, None


def _lined_up(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis.  ``weight`` and ``bias`` are of
    x's type or float32, and either may be missing."""
    code = _type(x, "layer_norm")
    types = (code, _param_type(x, weight, bias, code))
    if _recorded(x, weight, bias):
        return LayerNormFunction.apply(x, weight, bias, float(eps), types)
    return _norm(x, _lined_up(weight), _lined_up(bias), float(eps), types, False)[0]


# ---- the join ----------------------------------------------------------------------------------


def _add_norm(x, residual, weight, bias, p: float, state, eps: float, types, keep: bool):
    y, s = _new(x), _new(x)
    x, rows, width, ld = _rows(x)
    residual, _, _, ldr = _rows(residual)
    stats, mean, rstd = _stats(x, rows) if keep else (None, None, None)
    _lib.run(x.device, "zp_add_layernorm_forward", rows, width, types[0], x.data_ptr(), ld, residual.data_ptr(), ldr,
             p, _ptr(state), types[1], _ptr(weight), _ptr(bias), eps, s.data_ptr(), y.data_ptr(), mean, rstd)
    return y, s, stats


class DropoutAddLayerNormFunction(torch.autograd.Function):
    """``dropout_add_layer_norm`` with its gradients; ``state`` None: nothing is dropped."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, p: float, state, eps: float, types):
        weight, bias = _lined_up(weight), _lined_up(bias)
        y, s, stats = _add_norm(x, residual, weight, bias, p, state, eps, types, True)
        ctx.p, ctx.types = p, types
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(s, weight, bias, stats, state)
        return y, s

    @staticmethod
    @_first_order
    def backward(ctx, grad_y, grad_s):
        s, weight, bias, stats, state = ctx.saved_tensors
        want_x, want_res, want_w, want_b = ctx.needs_input_grad[:4]
        if grad_y is None and grad_s is None:
            return (None,) * 8
        _, rows, width, _ = _rows(s)
        dy, ldy = (None, 0) if grad_y is None else _rows(grad_y)[::3]
        ds, lds = (None, 0) if grad_s is None else _rows(grad_s)[::3]
        # without dropout the two gradients are one, and one tensor
        dres = torch.empty_like(s) if want_res or want_x and state is None else None
        dx = torch.empty_like(s) if want_x and state is not None else None
        dw, db, work, nbytes = _param_grads(weight, bias, want_w, want_b, rows)
        at = stats.data_ptr()
        _lib.run(s.device, "zp_add_layernorm_backward", rows, width, ctx.types[0], s.data_ptr(), ctx.types[1],
                 _ptr(weight), at, at + 4 * rows, _ptr(dy), ldy, _ptr(ds), lds, ctx.p, _ptr(state), _ptr(dx), _ptr(dres),
                 _ptr(dw), _ptr(db), _ptr(work), nbytes)
        return (dres if state is None and want_x else dx, dres if want_res else None, dw, db, None, None, None, None)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, p: float = 0.0,
                           state: torch.Tensor | None = None, eps: float = 1e-5):
    """``(y, s)``: ``s = residual + dropout(x, p, state)``, rounded to x's type, and
    ``y = layer_norm(s, weight, bias, eps)`` of s as it is returned, in one pass each way.  ``p = 0``
    (evaluation): no state is needed."""
    code = _type(x, "dropout_add_layer_norm")
    types = (code, _param_type(x, weight, bias, code))
    if residual.shape != x.shape:
        raise ValueError(f"the residual has shape {tuple(residual.shape)}, x {tuple(x.shape)}")
    if residual.get_device() != x.get_device():
        raise RuntimeError(f"the residual is on {residual.device}, x on {x.device}")
    if residual.dtype != x.dtype:
        raise TypeError(f"the residual is {residual.dtype}, x is {x.dtype}")
    if _threshold(p) == 0:
        p, state = 0.0, None
    else:
        _need_state(x, state)
    if _recorded(x, residual, weight, bias):
        return DropoutAddLayerNormFunction.apply(x, residual, weight, bias, float(p), state, float(eps), types)
    return _add_norm(x, residual, _lined_up(weight), _lined_up(bias), float(p), state, float(eps), types, False)[:2]


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
