"""Layer norm, dropout and their residual join on the GPU against the FP64 oracle.

Tolerances (u = 2^-24, a rounding in fp32; U v: a rounding to the result's type, eps / 2 of |v|, or of
the type's smallest normal number where |v| is smaller: below that the steps no longer shrink, in fp16
2^-24 under 2^-14, and half a step is 2^-25 = 2^-11 2^-14).  A sum of n terms of which
each is touched by at most D additions is off by D u times the sum of the magnitudes.  Along a row
D <= n / 32 + 32 (a lane's share of a row at least 32 lanes wide, and the steps that join the lanes;
a row of fewer than 32 lanes has at most 32 additions); over rows D <= n / 32 + 320.
    z = (x - mean) rstd    dz = rstd (D u mean|x| + 2 u |x|) + |z| (D + 6) u  (+ the mean's own error
                           enters the variance in second order only)
    y = z w + b            |w| dz + 2 u (|z w| + |b|) + U |y|
    gx = rstd (gz - m1 - z m2)   with errors of the sums m1, m2 of D u mean|gz|, D u mean|gz z| + mean(|gz| dz),
                           of z dz |m2|, and 6 u for the line itself; + U |gx|
    gw = sum gy z          D u sum|gy z| + sum(|gy| dz) + U |gw|
"""

from __future__ import annotations

import pytest
import torch

from oracle import rowwise_oracle as orc

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
u = 2.0 ** -24
EPS = 1e-5


def rowwise():
    from zippel_b200.blocks import rowwise as module
    return module


def near(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, what
    off = (got - want).abs() - tol
    assert not bool((off > 0).any()) and not bool(got.isnan().any()), (what, off.max().item())


def rounding(t, v):
    """The most that a value is off for being held in type t (half a step)."""
    info = torch.finfo(t)
    return v.abs().clamp_min(info.tiny) * (info.eps / 2)


def norm_case(rows, width, dtype, ptype, seed, affine=True, mean=0.3, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)             # noqa: E731
    x = (new(rows, width) * 1.5 + mean).to(dtype)
    gy, gs = new(rows, width).to(dtype), new(rows, width).to(dtype)
    w, b = ((1 + 0.3 * new(width)).to(ptype), (0.2 * new(width)).to(ptype)) if affine else (None, None)
    return x, w, b, gy, gs


class Want:
    """The oracle's results for rows x and the tolerances of the header."""

    def __init__(self, x, w, b, gy, dtype, ptype, gs=None):
        d = lambda t: None if t is None else t.double()                              # noqa: E731
        x, w, b, gy, gs = map(d, (x, w, b, gy, gs))
        r, n = x.shape
        D, Dr = n / 32 + 32, r / 32 + 320
        self.y, z, rstd = orc.layer_norm(x, w, b, EPS)
        self.gx, self.gw, self.gb = orc.layer_norm_vjp(z, rstd, w, gy)
        wa = torch.ones(n, dtype=torch.float64) if w is None else w.abs()
        ba = torch.zeros(n, dtype=torch.float64) if b is None else b.abs()
        mean = lambda t: t.mean(-1, keepdim=True)                                    # noqa: E731
        dz = rstd * (D * u * mean(x.abs()) + 2 * u * x.abs()) + z.abs() * (D + 6) * u
        self.ty = wa * dz + 2 * u * ((z * wa).abs() + ba) + rounding(dtype, self.y)
        gz = (gy * wa).abs()
        m2 = mean(gz * z.abs())
        line = rstd * (D * u * mean(gz) + z.abs() * (D * u * m2 + mean(gz * dz)) + dz * m2
                       + 6 * u * (gz + mean(gz) + z.abs() * m2))
        if gs is not None:
            self.gx = self.gx + gs
            line = line + 2 * u * gs.abs()
        self.line = line
        self.tgx = line + rounding(dtype, self.gx)
        self.tgw = Dr * u * (gy * z).abs().sum(0) + (gy.abs() * dz).sum(0) + rounding(ptype, self.gw)
        self.tgb = Dr * u * gy.abs().sum(0) + rounding(ptype, self.gb)


def up(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


WIDTHS = [1, 2, 7, 8, 31, 33, 100, 128, 255, 256, 257, 520, 1000, 1024, 1032, 2048, 2056, 4095, 4096, 4104, 8192,
          16384, 16392, 20011, 65544]


@pytest.mark.parametrize("dtype,ptype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("width", WIDTHS)
def test_layer_norm_and_gradients(width, dtype, ptype):
    for rows in (1, 3, 333) if width < 5000 else (1, 19):
        x, w, b, gy, _ = norm_case(rows, width, dtype, ptype, rows + width)
        want = Want(x, w, b, gy, dtype, ptype)
        xc, wc, bc, gc = up(x, w, b, gy)
        near(rowwise().layer_norm(xc, wc, bc, EPS), want.y, want.ty, "inference")
        leaves = [t.requires_grad_() for t in (xc, wc, bc)]
        y = rowwise().layer_norm(xc, wc, bc, EPS)
        gx, gw, gb = torch.autograd.grad(y, leaves, gc)
        near(y, want.y, want.ty, "y")
        near(gx, want.gx, want.tgx, "gx")
        near(gw, want.gw, want.tgw, "gw")
        near(gb, want.gb, want.tgb, "gb")
        assert y.dtype == gx.dtype == dtype and gw.dtype == gb.dtype == ptype


@pytest.mark.parametrize("dtype,rows,width", [(F32, 60000, 128), (BF16, 40001, 64), (F16, 5000, 1001), (BF16, 4999, 4096),
                                              (F32, 200003, 24)])
def test_layer_norm_of_many_rows(dtype, rows, width):
    x, w, b, gy, _ = norm_case(rows, width, dtype, dtype, 5)
    want = Want(x, w, b, gy, dtype, dtype)
    leaves = [t.requires_grad_() for t in up(x, w, b)]
    y = rowwise().layer_norm(*leaves, EPS)
    grads = torch.autograd.grad(y, leaves, gy.cuda(), retain_graph=True)
    near(y, want.y, want.ty)
    for got, ref, tol in zip(grads, (want.gx, want.gw, want.gb), (want.tgx, want.tgw, want.tgb)):
        near(got, ref, tol)
    again = torch.autograd.grad(y, leaves, gy.cuda())
    assert all(torch.equal(s, t) for s, t in zip(grads, again))          # fixed order of the sums


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [24, 33, 128, 4096])
def test_layer_norm_parameters_that_are_missing_or_frozen(width, dtype):
    x, w, b, gy, _ = norm_case(37, width, dtype, dtype, 3)
    xc, wc, bc, gc = up(x, w, b, gy)
    for weight, bias in ((None, None), (w, None), (None, b)):
        want = Want(x, weight, bias, gy, dtype, dtype)
        leaves = [xc.detach().requires_grad_()] + [t.cuda().requires_grad_() for t in (weight, bias) if t is not None]
        args = [leaves[0]] + [None if t is None else leaves[1] for t in (weight, bias)]
        y = rowwise().layer_norm(*args, EPS)
        near(y, want.y, want.ty)
        gx, *gp = torch.autograd.grad(y, leaves, gc)
        near(gx, want.gx, want.tgx)
        if gp:
            near(gp[0], *((want.gw, want.tgw) if weight is not None else (want.gb, want.tgb)))
    want = Want(x, w, b, gy, dtype, dtype)
    for on in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)):
        args = [t.detach().requires_grad_(bool(k)) for t, k in zip((xc, wc, bc), on)]
        y = rowwise().layer_norm(*args, EPS)
        got = torch.autograd.grad(y, [t for t in args if t.requires_grad], gc)
        refs = [(want.gx, want.tgx), (want.gw, want.tgw), (want.gb, want.tgb)]
        for g, r in zip(got, [r for r, k in zip(refs, on) if k]):
            near(g, *r)


def strided(x, kind):
    """x's values lying elsewhere than row behind row."""
    r, w = x.shape
    if kind == "rows":                       # rows of a wider array
        base = x.new_full((r, w + 24), float("nan"))
        base[:, 8:8 + w] = x
        return base[:, 8:8 + w]
    if kind == "odd":                        # rows that start at any address
        base = x.new_full((r, w + 3), float("nan"))
        base[:, 1:1 + w] = x
        return base[:, 1:1 + w]
    if kind == "offset":                     # contiguous, one element behind an aligned address
        base = x.new_full((r * w + 1,), float("nan"))
        base[1:] = x.reshape(-1)
        return base[1:].view(r, w)
    if kind == "transposed":
        return x.t().contiguous().t()
    raise KeyError(kind)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("kind", ["rows", "odd", "offset", "transposed"])
@pytest.mark.parametrize("width", [8, 33, 128, 1000, 4096])
def test_rows_that_lie_elsewhere(width, kind, dtype):
    x, w, b, gy, gs = norm_case(29, width, dtype, dtype, 11)
    xc, wc, bc, gc, sc = up(x, w, b, gy, gs)
    want = Want(x, w, b, gy, dtype, dtype)
    leaves = [t.requires_grad_() for t in (strided(xc, kind), strided(wc[None], "offset")[0], bc)]
    y = rowwise().layer_norm(*leaves, EPS)
    near(y, want.y, want.ty)
    gx, gw, gb = torch.autograd.grad(y, leaves, strided(gc, kind))
    near(gx, want.gx, want.tgx)
    near(gw, want.gw, want.tgw)
    near(gb, want.gb, want.tgb)
    state = torch.tensor([7, 9], device="cuda")
    plain = rowwise().dropout(xc, 0.3, state)
    assert torch.equal(rowwise().dropout(strided(xc, kind), 0.3, state), plain)
    a = rowwise().dropout_add_layer_norm(xc, sc, wc, bc, 0.3, state, EPS)
    b2 = rowwise().dropout_add_layer_norm(strided(xc, kind), strided(sc, kind), wc, bc, 0.3, state, EPS)
    assert torch.equal(a[1], b2[1])
    want = Want(a[1].cpu(), w, b, gy, dtype, dtype)        # (of the sum: its values are not x's)
    near(a[0], want.y, want.ty)
    near(b2[0], want.y, want.ty)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("width", [12, 100, 1002, 4090, 5001, 8186, 8190, 9999, 12288, 16377, 32768, 33001])
def test_rows_that_share_pieces_of_memory(width, dtype):
    """Widths that eight does not divide, of every class modulo eight, row behind row and from an odd address, few
    rows (fewer than a cycle of eight) and more than there are blocks: gradients of the join with dropout."""
    for rows in (1, 5, 400) if width < 2000 else (3, 310):
        x, w, b, gy, gs = norm_case(rows, width, dtype, dtype, rows + width)
        state, p = torch.tensor([rows, width]), 0.3
        f = torch.ones(rows, width, dtype=torch.float64)
        f = rowwise().dropout(f.float().cuda(), p, state.cuda()).double().cpu()        # (tested by itself)
        xc, wc, bc, gc, sc = up(x, w, b, gy, gs)
        for lie in (lambda t: t, lambda t: strided(t, "offset")):
            leaves = [t.detach().requires_grad_() for t in (lie(xc), lie(sc), wc, bc)]
            y, s = rowwise().dropout_add_layer_norm(*leaves, p, state.cuda(), EPS)
            total = x.double() * f + gs.double()
            near(s, total, rounding(dtype, total) + 4 * u * ((x.double() * f).abs() + total.abs()))
            want = Want(s.detach().cpu(), w, b, gy, dtype, dtype, gs)
            near(y, want.y, want.ty)
            gx, gr, gw, gb = torch.autograd.grad([y, s], leaves, [lie(gc), lie(sc)])
            near(gr, want.gx, want.tgx)
            near(gx, want.gx * f, (want.line + 4 * u * want.gx.abs()) * f + rounding(dtype, want.gx * f))
            near(gw, want.gw, want.tgw)
            near(gb, want.gb, want.tgb)
            plain = Want(x, w, b, gy, dtype, dtype)
            leaves = [t.detach().requires_grad_() for t in (lie(xc), wc, bc)]
            y = rowwise().layer_norm(*leaves, EPS)
            near(y, plain.y, plain.ty)
            for got, ref, tol in zip(torch.autograd.grad(y, leaves, lie(gc)), (plain.gx, plain.gw, plain.gb),
                                     (plain.tgx, plain.tgw, plain.tgb)):
                near(got, ref, tol)


def test_neighbours_of_a_result_stay_as_they_are():
    """Results of odd rows in the middle of an array, through the C ABI: what lies before and behind is not
    touched, nor what the rows do not cover."""
    from zippel_b200 import _lib
    for rows, width, code, dt in ((9, 33, 0, F32), (9, 1001, 1, F16), (3, 7, 2, BF16), (300, 9, 1, F16)):
        for lead in (0, 8, 16, 3):
            x = torch.randn(rows, width, device="cuda").to(dt)
            n = rows * width
            y, s, stats = (torch.full((n + 64,), -7.0, device="cuda", dtype=dt) for _ in range(3))
            stats = torch.empty(2, rows, device="cuda")
            size = dt.itemsize
            _lib.run(x.device, "zp_add_layernorm_forward", rows, width, code, x.data_ptr(), width, x.data_ptr(), width, 0.0,
                     None, code, None, None, 1e-5, s.data_ptr() + lead * size, y.data_ptr() + lead * size,
                     stats.data_ptr(), stats.data_ptr() + 4 * rows)
            for t, ref in ((s, x + x), (y, torch.nn.functional.layer_norm((x + x).double(), (width,)).to(dt))):
                assert bool((t[:lead] == -7).all()) and bool((t[lead + n:] == -7).all())
                assert (t[lead:lead + n].view(rows, width).double() - ref.double()).abs().max() < 0.02


def test_leading_axes():
    x, w, b, gy, _ = norm_case(4 * 6, 40, F32, F32, 1)
    want = Want(x, w, b, gy, F32, F32)
    shaped = lambda t: t.view(4, 6, 40)                                             # noqa: E731
    xc, wc, bc, gc = up(x, w, b, gy)
    base = torch.zeros(4, 6, 3, 40, device="cuda")
    base[:, :, 1] = shaped(xc)
    for v in (shaped(xc), base[:, :, 1], shaped(xc).transpose(0, 1).contiguous().transpose(0, 1)):
        leaf = v.detach().requires_grad_()
        y = rowwise().layer_norm(leaf, wc, bc, EPS)
        near(y, shaped(want.y), shaped(want.ty))
        near(torch.autograd.grad(y, leaf, shaped(gc))[0], shaped(want.gx), shaped(want.tgx))
    # a gradient that is one number everywhere
    leaf = xc.detach().requires_grad_()
    ones = Want(x, w, b, torch.ones_like(gy), F32, F32)
    near(torch.autograd.grad(rowwise().layer_norm(leaf, wc, bc, EPS).sum(), leaf)[0], ones.gx, ones.tgx)
    near(rowwise().layer_norm(xc[0], wc, bc, EPS), want.y[0], want.ty[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_far_from_zero_equal_or_not_finite(dtype):
    """A row of equal values has y = bias; a mean 1000 times the spread loses 2^-24 of it, no more; NaN
    and infinities stay in their rows."""
    g = torch.Generator().manual_seed(2)
    for width in (33, 128, 1024, 4096):
        x = torch.randn(8, width, generator=g, dtype=torch.float64)
        x[1] = 3.0
        x[2] += 1000.0
        x[3] *= 1e-4
        x[4] *= 1e4
        x[6, 1], x[7, 0] = float("inf"), float("nan")
        x = x.to(dtype)
        w, b = (torch.randn(width, generator=g, dtype=torch.float64).to(dtype) for _ in range(2))
        want = Want(x[:6], w, b, torch.ones(6, width, dtype=dtype), dtype, dtype)
        y = rowwise().layer_norm(*up(x, w, b), EPS)
        near(y[:6], want.y, want.ty)
        assert torch.equal(y[1].cpu(), b)
        assert bool(y[6:].isnan().all())


@pytest.mark.parametrize("width", [5, 33, 65, 100, 104, 120, 129, 200])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("extra", [0, 1])
def test_gradients_of_equal_rows_of_large_values(dtype, width, extra):
    """Rows of 2^120: their sums are exact, width times fp32(1 / width) is 1 for these widths, so that z is 0 and
    gx = rstd (gz - mean gz), gw = 0, though mean times rstd is past fp32."""
    g = torch.Generator().manual_seed(3)
    gy = torch.randn(20, width, generator=g, dtype=torch.float64).to(dtype)
    w = (1 + 0.3 * torch.randn(width, generator=g, dtype=torch.float64)).to(dtype)
    gz = gy.double() * w.double()
    m = gz.abs().mean(-1, keepdim=True)
    want = (gz - gz.mean(-1, keepdim=True)) * EPS ** -0.5
    tol = EPS ** -0.5 * ((width / 32 + 32) * u * m + 6 * u * (gz.abs() + m)) + rounding(dtype, want)
    base = torch.full((20, width + extra), 2.0 ** 120, dtype=dtype, device="cuda")
    wc, gc = up(w, gy)
    x, wc = base[:, :width].detach().requires_grad_(), wc.requires_grad_()
    rw = rowwise()
    grads = torch.autograd.grad(rw.layer_norm(x, wc, torch.zeros_like(wc), EPS), (x, wc), gc)
    near(grads[0], want, tol, "norm")
    assert not bool(grads[1].any())
    zero = torch.zeros_like(x)
    y, _ = rw.dropout_add_layer_norm(zero, x, wc, torch.zeros_like(wc), 0.0, None, EPS)
    near(torch.autograd.grad(y, x, gc)[0], want, tol, "join")


def test_no_rows_and_refusals():
    rw = rowwise()
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    b = torch.ones(16, device="cuda", requires_grad=True)
    y, s = rw.dropout_add_layer_norm(x, x, w, b, 0.5, rw.dropout_state("cuda"))
    assert y.shape == s.shape == (0, 16)
    for t in (y.sum() + s.sum(), rw.layer_norm(x, w, b).sum()):
        gx, gw, gb = torch.autograd.grad(t, [x, w, b])
        assert gx.shape == (0, 16) and not gw.any() and not gb.any()
    assert rw.dropout(x, 0.5, rw.dropout_state("cuda")).shape == (0, 16)
    assert rw.dropout(torch.zeros(3, 0, device="cuda"), 0.5, rw.dropout_state("cuda")).shape == (3, 0)
    x, st = torch.zeros(4, 16, device="cuda"), rw.dropout_state("cuda")
    assert rw.dropout(x, 0.0) is x and rw.dropout(x, 1e-6) is x
    bad = [(ValueError, lambda: rw.layer_norm(x, torch.ones(8, device="cuda"))),
           (ValueError, lambda: rw.layer_norm(x, bias=torch.ones(1, device="cuda"))),
           (TypeError, lambda: rw.layer_norm(x, torch.ones(16, device="cuda", dtype=F16))),
           (TypeError, lambda: rw.layer_norm(x.half(), torch.ones(16, device="cuda"), torch.ones(16, device="cuda", dtype=F16))),
           (TypeError, lambda: rw.layer_norm(x.double())), (RuntimeError, lambda: rw.layer_norm(x, torch.ones(16))),
           (ValueError, lambda: rw.layer_norm(torch.zeros((), device="cuda"))),
           (ValueError, lambda: rw.layer_norm(torch.zeros(3, 0, device="cuda"))),
           (ValueError, lambda: rw.dropout(x, 1.5, st)), (ValueError, lambda: rw.dropout(x, 0.5)),
           (ValueError, lambda: rw.dropout(x, float("nan"), st)),
           (ValueError, lambda: rw.dropout(x, 0.5, st.int())), (ValueError, lambda: rw.dropout(x, 0.5, st[:1])),
           (RuntimeError, lambda: rw.dropout(x, 0.5, st.cpu())), (TypeError, lambda: rw.dropout(x.long(), 0.5, st)),
           (ValueError, lambda: rw.dropout_add_layer_norm(x, x[:1])), (TypeError, lambda: rw.dropout_add_layer_norm(x, x.half())),
           (RuntimeError, lambda: rw.dropout_add_layer_norm(x, x.cpu())),
           (ValueError, lambda: rw.dropout_add_layer_norm(x, x, p=0.5))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5), (16, 128), (29, 1001), (2, 3, 4096), ()])
@pytest.mark.parametrize("p", [0.1, 0.5, 1.0, 2.0 ** -16])
def test_dropout_and_gradient(shape, dtype, p):
    """Which elements are kept, bit for bit; the factor is off by a rounding of itself and one of the
    product, beside the result's own."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)
    gy = torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)
    state = torch.tensor([-2 ** 62 + 12345, 2 ** 40 + 3], dtype=torch.int64)
    f = orc.factors(shape, p, state.tolist())
    xc = x.cuda().requires_grad_()
    y = rowwise().dropout(xc, p, state.cuda())
    gx, = torch.autograd.grad(y, xc, gy.cuda())
    for got, v in ((y, x), (gx, gy)):
        want = v.double() * f
        near(got, want, rounding(dtype, want) + 3 * u * want.abs())
        assert torch.equal(got.cpu() == 0, (f == 0) | (v == 0))
    plain = rowwise().dropout(x.cuda(), p, state.cuda())
    assert torch.equal(plain, y)


def test_dropout_leaves_nothing_of_what_it_drops_and_nothing_between_the_rows():
    from zippel_b200 import _lib
    state = torch.tensor([5, 6], device="cuda")
    f = orc.factors((4, 24), 0.5, (5, 6)).cuda()
    x = torch.where(f == 0, float("nan"), 2.0)
    x[0] = torch.where(f[0] == 0, float("inf"), 2.0)
    y = rowwise().dropout(x, 0.5, state)
    assert torch.equal(y, torch.where(f == 0, 0.0, 4.0))
    for width in (24, 21):
        out = torch.full((4, 32), -7.0, device="cuda")
        _lib.run(x.device, "zp_dropout", 4, width, 0, x.data_ptr(), 24, 0.5, state.data_ptr(), out.data_ptr(), 32)
        assert bool((out[:, width:] == -7).all()) and bool((out[:, :width] != -7).all())


def test_element_numbers_past_32_bits():
    """2^32 + 64 elements in fp16 (8.6 GB): the last ones and those around the border, by the counter's
    upper word."""
    n = 2 ** 32 + 64
    state = torch.tensor([11, 13], device="cuda")
    x = torch.ones(n, dtype=F16, device="cuda")
    y = rowwise().dropout(x, 0.5, state)
    del x
    for first in (0, 2 ** 31 - 64, 2 ** 32 - 64, 2 ** 32):
        assert torch.equal(y[first:first + 64].cpu() != 0, orc.kept(64, 0.5, (11, 13), first))
    del y


def test_rows_past_32_bits():
    """More than 2^32 elements (8.6 GB an array): rows on either side of the border, forward and backward."""
    rows, width = 2 ** 20 + 64, 4096
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.empty(rows, width, device="cuda", dtype=BF16).normal_(generator=g).requires_grad_()
    gy = torch.empty(rows, width, device="cuda", dtype=BF16).normal_(generator=g)
    y = rowwise().layer_norm(x, None, None, EPS)
    gx, = torch.autograd.grad(y, x, gy)
    for first in (0, 2 ** 19 - 4, 2 ** 20 - 4, rows - 8):
        part = slice(first, first + 8)
        want = Want(x.detach()[part].cpu(), None, None, gy[part].cpu(), BF16, BF16)
        near(y[part], want.y, want.ty)
        near(gx[part], want.gx, want.tgx)


@pytest.mark.parametrize("dtype,width", [(F32, 128), (F32, 33), (BF16, 4096), (BF16, 520), (F16, 1001), (F16, 7),
                                         (BF16, 16384), (F32, 20011)])
@pytest.mark.parametrize("p", [0.0, 0.25, 1.0])
def test_join_and_gradients(dtype, width, p):
    """s against one rounding of the exact sum; y and the gradients against the oracle's for s as it was
    returned."""
    for rows in (1, 45):
        x, w, b, gy, gs = norm_case(rows, width, dtype, dtype, rows + width)
        res = torch.randn(rows, width, generator=torch.Generator().manual_seed(9), dtype=torch.float64).to(dtype)
        state = torch.tensor([rows, width], dtype=torch.int64)
        f = orc.factors((rows, width), p, state.tolist())
        xc, rc, wc, bc, gc, sc = up(x, res, w, b, gy, gs)
        st = state.cuda() if p else None
        plain = rowwise().dropout_add_layer_norm(xc, rc, wc, bc, p, st, EPS)
        leaves = [t.requires_grad_() for t in (xc, rc, wc, bc)]
        y, s = rowwise().dropout_add_layer_norm(*leaves, p, st, EPS)
        assert torch.equal(plain[0], y) and torch.equal(plain[1], s)
        total = x.double() * f + res.double()
        near(s, total, rounding(dtype, total) + 3 * u * ((x.double() * f).abs() + total.abs()))
        for up_y, up_s in ((gc, sc), (gc, None), (None, sc)):
            want = Want(s.detach().cpu(), w, b, gy if up_y is not None else torch.zeros_like(gy), dtype, dtype,
                        gs if up_s is not None else None)
            near(y, want.y, want.ty)
            outs = [t for t, k in ((y, up_y), (s, up_s)) if k is not None]
            gx, gr, gw, gb = torch.autograd.grad(outs, leaves, [t for t in (up_y, up_s) if t is not None],
                                                 retain_graph=True)
            near(gr, want.gx, want.tgx)
            near(gx, want.gx * f, (want.line + 3 * u * want.gx.abs()) * f + rounding(dtype, want.gx * f))
            assert torch.equal(gx.cpu() == 0, (gr.cpu() == 0) | (f == 0))
            near(gw, want.gw, want.tgw)
            near(gb, want.gb, want.tgb)
        for k in range(4):                     # each gradient by itself
            one = [t.detach().requires_grad_(j == k) for j, t in enumerate(leaves)]
            y1, s1 = rowwise().dropout_add_layer_norm(*one, p, st, EPS)
            g1, = torch.autograd.grad([y1] if k > 1 else [y1, s1], [one[k]], [gc] if k > 1 else [gc, sc])
            full = torch.autograd.grad([y, s], leaves, [gc, sc], retain_graph=True)[k]
            assert torch.equal(g1, full)


def test_gradients_against_differences():
    """Central differences of the fp32 kernels along one direction per input: with steps of 2^-6 in 64
    rows of 96 the truncation is of order h^2 = 2.4e-4 of the third derivative, the rounding
    2^-24 sqrt(6144) / h = 3e-4; a third of a per cent of the gradient's own size holds both."""
    g = torch.Generator("cuda").manual_seed(4)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")                    # noqa: E731
    ins = [new(64, 96), new(64, 96), 1 + 0.2 * new(96), new(96)]
    gy, gs, st = new(64, 96), new(64, 96), torch.tensor([3, 4], device="cuda")

    def value(ts):
        y, s = rowwise().dropout_add_layer_norm(*ts, 0.2, st, EPS)
        return (y.double() * gy.double()).sum() + (s.double() * gs.double()).sum()

    leaves = [t.clone().requires_grad_() for t in ins]
    grads = torch.autograd.grad(value(leaves), leaves)
    for i, (t, grad) in enumerate(zip(ins, grads)):
        d = new(*t.shape)
        h = 2.0 ** -6
        f = [value([v + k * h * d if j == i else v for j, v in enumerate(ins)]) for k in (1, -1)]
        slope = ((f[0] - f[1]) / (2 * h)).item()
        size = grad.norm().item() * d.norm().item() / d.numel() ** 0.5
        assert abs(slope - (grad.double() * d.double()).sum().item()) < size / 300, i


def test_side_stream_capture_and_new_states():
    """A training pass of all three on another stream, recorded and replayed: replays follow what lies in
    the inputs and in the state."""
    rw = rowwise()
    x, w, b, gy, gs = up(*norm_case(70, 136, F32, F32, 8))
    state = torch.tensor([1, 2], device="cuda")

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        h = rw.dropout(rw.layer_norm(*leaves, EPS), 0.3, state)
        y, s = rw.dropout_add_layer_norm(h, leaves[0], leaves[1], leaves[2], 0.2, state, EPS)
        return [y, s, *torch.autograd.grad([y, s], leaves, [gy, gs])]

    first = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.detach().clone() for t in step()]
        side.synchronize()
        assert all(torch.equal(s, t) for s, t in zip(first, other))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(s, t) for s, t in zip(first, out))
    state.copy_(torch.tensor([5, 2], device="cuda"))
    x.mul_(1.5)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in out]
    want = step()
    assert all(torch.equal(s, t) for s, t in zip(want, got)) and not torch.equal(got[0], first[0])


def test_a_state_drawn_while_recording_is_new_in_every_replay():
    rw = rowwise()
    x = torch.ones(64, 64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rw.dropout(x, 0.5, rw.dropout_state("cuda"))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = rw.dropout(x, 0.5, rw.dropout_state("cuda"))
    seen = []
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(y.clone())
    assert not torch.equal(*seen) and abs(seen[0].mean().item() - 1) < 0.1


def test_inputs_changed_before_the_backward_are_noticed():
    rw = rowwise()
    x, w, b, gy, _ = up(*norm_case(8, 32, F32, F32, 8))
    leaf, state = x.clone().requires_grad_(), rw.dropout_state("cuda")
    y = rw.dropout(leaf, 0.5, state)
    state.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y, leaf, gy)
    with pytest.raises(RuntimeError):          # first order only
        g, = torch.autograd.grad(rw.layer_norm(leaf, w, b), leaf, gy, create_graph=True)
        torch.autograd.grad(g.sum(), leaf)


def test_nothing_dropped_through_the_c_abi_copies():
    from zippel_b200 import _lib
    state = torch.tensor([5, 6], device="cuda")
    x = torch.randn(5, 12, device="cuda")
    for width, ldy in ((12, 12), (12, 20), (7, 7)):
        y = torch.full((5, ldy), -7.0, device="cuda")
        _lib.run(x.device, "zp_dropout", 5, width, 0, x.data_ptr(), 12, 0.0, state.data_ptr(), y.data_ptr(), ldy)
        assert torch.equal(y[:, :width], x[:, :width]) and bool((y[:, width:] == -7).all())


def test_calls_that_torch_wraps():
    """Tangents and batched tensors are refused, not read past; inference tensors and gradients of the same
    tensor given twice are served."""
    import torch.autograd.forward_ad as fwd
    rw = rowwise()
    x, w, b, gy, _ = up(*norm_case(8, 32, F32, F32, 8))
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        rw.layer_norm(fwd.make_dual(x, gy), w, b)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda v: rw.layer_norm(v, w, b))(x.view(2, 4, 32))
    with torch.inference_mode():
        y = rw.layer_norm(x, w, b)
        z, s = rw.dropout_add_layer_norm(x, x, w, b, 0.5, rw.dropout_state("cuda"))
    assert torch.equal(y, rw.layer_norm(x, w, b)) and not y.requires_grad and z.shape == s.shape
    leaf = x.clone().requires_grad_()
    y, s = rw.dropout_add_layer_norm(leaf, leaf, w, b)
    twice, = torch.autograd.grad(y, leaf, gy)
    pair = [x.clone().requires_grad_() for _ in range(2)]
    one, other = torch.autograd.grad(rw.dropout_add_layer_norm(*pair, w, b)[0], pair, gy)
    assert torch.equal(twice, one + other)


def test_two_streams_and_threads_at_once():
    """The same leaves through forward and backward on two streams from two threads, many times: no scratch is
    shared."""
    import threading
    rw = rowwise()
    cases = [up(*norm_case(300, width, F32, F32, width)) for width in (1001, 4096)]
    state = torch.tensor([1, 2], device="cuda")

    def work(case):
        x, w, b, gy, gs = case
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y, s = rw.dropout_add_layer_norm(leaves[0], gs, leaves[1], leaves[2], 0.3, state)
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], leaves, [gy, gs])]

    want = [work(c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                got = work(cases[i])
                stream.synchronize()
                if not all(torch.equal(a, c) for a, c in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1, 0)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad
