"""Rows of equal values whose sums are exact: their mean is the value, z is 0, y is the bias and the gradient of the rows
rstd (gz - mean gz), at widths of which one over the width is not what its float says."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_rowwise import BF16, EPS, F16, F32, near, rounding, rowwise, u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [3, 7, 41, 47, 55, 61, 82, 83, 97, 1000, 1001, 1025, 4001, 4090, 9999, 16388, 20011])
@pytest.mark.parametrize("extra", [0, 1])
def test_rows_of_equal_values_of_exact_sums(width, dtype, extra):
    """Values of eight bits at most (768 and 1000: 1.5 and 1.953125 times a power of two) and 32 767 columns at most: every
    sum on the way is a whole number below 2^24 times a power of two, whatever the order.  gx as in the
    oracle's tolerances, with z 0: rstd (D u mean|gz| + 6 u (|gz| + mean|gz|)) and the result's own rounding."""
    g = torch.Generator().manual_seed(width)
    new = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)    # noqa: E731
    values = torch.tensor([1000.0, 3.0, 768.0, -1000.0, 0.0, 2.0 ** -10])
    gy, w, b = new(len(values), width), new(width), new(width)
    gz = gy.double() * w.double()
    m = gz.abs().mean(-1, keepdim=True)
    want = (gz - gz.mean(-1, keepdim=True)) * EPS ** -0.5
    tol = EPS ** -0.5 * ((width / 32 + 32) * u * m + 6 * u * (gz.abs() + m)) + rounding(dtype, want)
    base = values[:, None].expand(-1, width + extra).to(dtype).cuda()
    base = base.contiguous()
    x = base[:, :width].detach().requires_grad_()
    wc, bc, gc = w.cuda().requires_grad_(), b.cuda().requires_grad_(), gy.cuda()
    rw = rowwise()
    y = rw.layer_norm(x, wc, bc, EPS)
    assert torch.equal(y, bc.expand_as(y))
    gx, gw = torch.autograd.grad(y, (x, wc), gc)
    near(gx, want, tol, "norm")
    assert not gw.any()
    zero = torch.zeros_like(x)
    y, s = rw.dropout_add_layer_norm(zero, x, wc, bc, 0.0, None, EPS)
    assert torch.equal(s, x) and torch.equal(y, bc.expand_as(y))
    gx, gw = torch.autograd.grad(y, (x, wc), gc)
    near(gx, want, tol, "join")
    assert not gw.any()
