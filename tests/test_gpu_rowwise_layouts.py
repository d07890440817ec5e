"""Layer norm, dropout and their join of tensors whose rows are one row repeated, or overlap, as inputs and as
upstream gradients: what the same calls give for dense copies of them, and sums over rows against the FP64 oracle."""

from __future__ import annotations

import pytest
import torch

from oracle import rowwise_oracle as orc
from tests.test_gpu_rowwise import EPS, F16, F32, Want, near, norm_case, rounding, rowwise, u, up

pytestmark = pytest.mark.gpu

SHAPE = (3, 20)                               # of the leading axes


def repeated(kind, width, dtype, seed):
    """A tensor [3, 20, width] over a storage of fewer elements."""
    g = torch.Generator("cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)          # noqa: E731
    if kind == "one row":
        return new(width).expand(*SHAPE, width)
    if kind == "rows inside":
        return new(SHAPE[0], 1, width).expand(*SHAPE, width)
    if kind == "rows outside":
        return new(1, SHAPE[1], width).expand(*SHAPE, width)
    if kind == "one number":
        return new(1, 1, 1).expand(*SHAPE, width)
    if kind == "overlapping":
        return new(2 * width + SHAPE[0] * 40 + SHAPE[1] * 2).as_strided((*SHAPE, width), (40, 2, 1))
    raise KeyError(kind)


KINDS = ["one row", "rows inside", "rows outside", "one number", "overlapping"]


def same(got, want, gy):
    """Equal bit for bit, but for gradients of weight and bias of width 1: rows of one number in steps of two or forty do
    not overlap and are read where they lie, by other teams, so sums over rows are taken in another order.  Two orders
    of n terms differ by twice (n / 32 + 320) u times the sum of the magnitudes and a rounding each; the weight's
    terms are zero (a row of one has z = 0)."""
    for (name, g), (_, ref) in zip(got, want, strict=True):
        if g.shape == (1,):
            rows = gy.numel()
            near(g, ref.cpu(), (2 * (rows / 32 + 320) * u * gy.double().abs().sum() + 2 * rounding(g.dtype, ref.double())).cpu(), name)
        else:
            assert torch.equal(g, ref), name


def calls(x, res, w, b, gy, gs):
    """All three operators' results and gradients."""
    rw, state, out = rowwise(), torch.tensor([5, 6], device="cuda"), []
    for name, f in (("norm", lambda t, r, *wb: [rw.layer_norm(t, *wb, EPS)]),
                    ("dropout", lambda t, r, *wb: [rw.dropout(t, 0.3, state)]),
                    ("join", lambda t, r, *wb: rw.dropout_add_layer_norm(t, r, *wb, 0.3, state, EPS)),
                    ("join without dropout", lambda t, r, *wb: rw.dropout_add_layer_norm(t, r, *wb, 0.0, None, EPS))):
        with torch.no_grad():
            out += [(name, t) for t in f(x, res, w, b)]
        leaves = [t.detach().requires_grad_() for t in (x, res, w, b)]
        ys = list(f(*leaves))
        grads = torch.autograd.grad(ys, leaves, [gy, gs][:len(ys)], allow_unused=True)
        out += [(name, t) for t in (*ys, *grads) if t is not None]
    return out


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("width", [1, 33, 128])
def test_repeated_rows_as_their_copies(width, kind, dtype):
    t = [repeated(kind, width, dtype, seed) for seed in range(4)]
    w, b = repeated("one row", width, dtype, 8)[0, 0], repeated("one row", width, dtype, 9)[0, 0]
    assert not any(v.is_contiguous() for v in t)
    want = calls(t[0].contiguous(), t[1].contiguous(), w, b, t[2].contiguous(), t[3].contiguous())
    for where in range(4):                     # one of x, residual and the gradients, and all
        args = [v if i == where else v.contiguous() for i, v in enumerate(t)]
        same(calls(args[0], args[1], w, b, args[2], args[3]), want, t[2])
    same(calls(t[0], t[1], w, b, t[2], t[3]), want, t[2])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("width", [1, 24, 33, 128])
@pytest.mark.parametrize("over", [0, 1, (0, 1)])
def test_gradients_of_sums_over_rows(over, width, dtype):
    """The gradient of (sum of rows * v): every row's upstream gradient is v, or one of a few."""
    rows = SHAPE[0] * SHAPE[1]
    x, w, b, _, res = norm_case(rows, width, dtype, dtype, width)
    v = torch.zeros(*SHAPE, width, dtype=torch.float64).sum(over)
    v = torch.randn(v.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64).to(dtype)
    axes = (over,) if isinstance(over, int) else over
    dense = v
    for a in axes:
        dense = dense.unsqueeze(a)
    gy = dense.expand(*SHAPE, width).reshape(rows, width)
    xc, wc, bc, rc, vc = up(x.view(*SHAPE, width), w, b, res.view(*SHAPE, width), v)
    rw, state = rowwise(), torch.tensor([5, 6], device="cuda")
    f = orc.factors((rows, width), 0.3, (5, 6))

    leaves = [t.clone().requires_grad_() for t in (xc, wc, bc)]
    got = torch.autograd.grad(rw.layer_norm(*leaves, EPS).sum(over), leaves, vc)
    want = Want(x, w, b, gy, dtype, dtype)
    for g, ref, tol in zip(got, (want.gx.view(*SHAPE, width), want.gw, want.gb),
                           (want.tgx.view(*SHAPE, width), want.tgw, want.tgb)):
        near(g, ref, tol, "norm")

    leaf = xc.clone().requires_grad_()
    g, = torch.autograd.grad(rw.dropout(leaf, 0.3, state).sum(over), leaf, vc)
    ref = gy.double() * f
    near(g.view(rows, width), ref, rounding(dtype, ref) + 3 * u * ref.abs(), "dropout")

    leaves = [t.clone().requires_grad_() for t in (xc, rc, wc, bc)]
    y, s = rw.dropout_add_layer_norm(*leaves, 0.3, state, EPS)
    got = torch.autograd.grad([y.sum(over), s.sum(over)], leaves, [vc, vc])
    want = Want(s.detach().cpu().view(rows, width), w, b, gy, dtype, dtype, gy)
    near(got[1].view(rows, width), want.gx, want.tgx, "residual")
    near(got[0].view(rows, width), want.gx * f, (want.line + 3 * u * want.gx.abs()) * f + rounding(dtype, want.gx * f), "x")
    near(got[2], want.gw, want.tgw, "weight")
    near(got[3], want.gb, want.tgb, "bias")


@pytest.mark.parametrize("width", [1, 24])
def test_lazy_negations_and_zeroes(width):
    """Rows, parameters and gradients whose values are not what lies in memory."""
    g = torch.Generator("cuda").manual_seed(1)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")                    # noqa: E731
    if width == 1:
        lazy = [torch.complex(new(*s), new(*s)).conj().imag for s in [(40, 1)] * 4 + [(1,)] * 2]
    else:
        lazy = [torch._neg_view(new(*s)) for s in [(40, width)] * 4 + [(width,)] * 2]
    assert all(t.is_neg() for t in lazy)
    order = lambda t: (t[0], t[1], t[4], t[5], t[2], t[3])                          # noqa: E731
    plain = [t.clone(memory_format=torch.contiguous_format) for t in lazy]
    assert not any(t.is_neg() for t in plain)
    same(calls(*order(lazy)), calls(*order(plain)), plain[2])

    leaves = [t.clone().requires_grad_() for t in (plain[0], plain[1])]
    ys = rowwise().dropout_add_layer_norm(*leaves, None, None, 0.3, torch.tensor([5, 6], device="cuda"))
    zero = torch._efficientzerotensor((40, width), device="cuda")
    got = torch.autograd.grad(ys, leaves, [zero, plain[3]], retain_graph=True)
    want = torch.autograd.grad(ys, leaves, [torch.zeros(40, width, device="cuda"), plain[3]])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
