"""Layer norm, dropout and their join, what needs no GPU: the oracle's generator against its published
vectors and its gradients against differences, and the refusals of the C ABI and of the Python layer."""

from __future__ import annotations

import pytest
import torch

from oracle import rowwise_oracle as orc

M = 0xFFFFFFFF


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((M, M, M, M), (M, M), (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))])
def test_generator_against_its_published_vectors(counter, key, want):
    assert tuple(orc.philox(counter, key)) == want


def test_share_that_is_kept():
    """4096 elements: the share dropped is within five standard deviations of p."""
    for p in (0.1, 0.5, 0.9):
        share = 1 - orc.kept(4096, p, (12345, 678)).double().mean().item()
        assert abs(share - p) < 5 * (p * (1 - p) / 4096) ** 0.5
    assert bool(orc.kept(64, 0.0, (1, 2)).all()) and not bool(orc.kept(64, 1.0, (1, 2)).any())


def test_oracle_gradients_against_differences():
    """Central differences in 64 bits: the truncation is h^2 / 6 times a third derivative of order ten,
    the rounding 2^-53 / h: 1e-8 with h = 1e-5 leaves room for both."""
    g = torch.Generator().manual_seed(0)
    new = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)             # noqa: E731
    x, w, b, gy = new(5, 7), new(7), new(7), new(5, 7)
    _, z, rstd = orc.layer_norm(x, w, b, 1e-5)
    grads = orc.layer_norm_vjp(z, rstd, w, gy)
    for i, t in enumerate((x, w, b)):
        d = new(*t.shape)
        h = 1e-5
        f = [(orc.layer_norm(*[v + s * h * d if j == i else v for j, v in enumerate((x, w, b))], 1e-5)[0]
              * gy).sum() for s in (1, -1)]
        assert abs(((f[0] - f[1]) / (2 * h) - (grads[i] * d).sum()).item()) < 1e-8


@pytest.fixture(scope="module")
def lib():
    from zippel_b200 import _lib, build
    build.build_library()
    return _lib.load()


A = 4096                                      # an address that is never read: arguments are looked at first


def test_refusals_of_the_c_abi(lib):
    drop = lambda rows=2, width=8, dtype=0, x=A, ldx=8, p=0.5, st=A, y=A, ldy=8: (          # noqa: E731
        lib.zp_dropout(rows, width, dtype, x, ldx, p, st, y, ldy, None))
    assert drop(rows=-1) == 1 and drop(width=0) == 1 and drop(dtype=3) == 2 and drop(dtype=-1) == 2
    assert drop(x=None) == 1 and drop(y=None) == 1 and drop(st=None) == 1 and drop(st=A + 4) == 1
    assert drop(ldx=7) == 1 and drop(ldy=7) == 1
    assert drop(p=-0.1) == 1 and drop(p=1.1) == 1 and drop(p=float("nan")) == 1
    assert drop(x=A + 2) == 1 and drop(dtype=1, x=A + 1) == 1
    assert drop(rows=2 ** 61, width=2 ** 10) == 2 and drop(rows=2 ** 31, ldx=2 ** 40) == 1
    assert drop(rows=0, x=None, y=None, st=None) == 0 and drop(rows=0, p=2.0) == 1

    fwd = lambda rows=2, width=8, dtype=0, x=A, ldx=8, pt=0, w=A, b=A, y=A, mean=A, rstd=A: (   # noqa: E731
        lib.zp_layernorm_forward(rows, width, dtype, x, ldx, pt, w, b, 1e-5, y, mean, rstd, None))
    assert fwd(rows=-1) == 1 and fwd(width=0) == 1 and fwd(dtype=7) == 2
    assert fwd(dtype=0, pt=1) == 2 and fwd(dtype=1, pt=2) == 2 and fwd(pt=9) == 2
    assert fwd(x=None) == 1 and fwd(y=None) == 1 and fwd(ldx=7) == 1
    assert fwd(mean=None) == 1 and fwd(rstd=None) == 1 and fwd(w=A + 2) == 1 and fwd(b=A + 1) == 1
    assert fwd(rows=0, x=None, y=None) == 0

    nbytes = lib.zp_rowwise_work_bytes(2, 8)
    assert nbytes >= 2 * 8 * 4 and lib.zp_rowwise_work_bytes(0, 8) == 0 and lib.zp_rowwise_work_bytes(2, 0) == 0
    bwd = lambda rows=2, width=8, dtype=0, x=A, pt=0, mean=A, rstd=A, dy=A, ldy=8, dw=A, work=A, nb=nbytes: (  # noqa: E731
        lib.zp_layernorm_backward(rows, width, dtype, x, 8, pt, A, mean, rstd, dy, ldy, A, dw, A, work, nb, None))
    assert bwd(rows=-1) == 1 and bwd(dtype=5) == 2 and bwd(pt=1) == 2
    assert bwd(x=None) == 1 and bwd(mean=None) == 1 and bwd(rstd=None) == 1 and bwd(dy=None) == 1
    assert bwd(ldy=7) == 1 and bwd(work=None) == 1 and bwd(nb=nbytes - 1) == 3 and bwd(dw=A + 2) == 1

    add = lambda rows=2, width=8, dtype=0, res=A, ldr=8, p=0.5, st=A, sum=A, y=A: (               # noqa: E731
        lib.zp_add_layernorm_forward(rows, width, dtype, A, 8, res, ldr, p, st, 0, A, A, 1e-5, sum, y, A, A, None))
    assert add(rows=-1) == 1 and add(dtype=3) == 2 and add(res=None) == 1 and add(ldr=7) == 1
    assert add(p=2.0) == 1 and add(st=None) == 1 and add(sum=None) == 1 and add(y=None) == 1
    assert add(rows=0, res=None) == 0 and add(rows=0, p=-1.0) == 1
    addb = lambda dtype=0, dy=A, dsum=A, lds=8, p=0.5, st=A, work=A: (                            # noqa: E731
        lib.zp_add_layernorm_backward(2, 8, dtype, A, 0, A, A, A, dy, 8, dsum, lds, p, st, A, A, A, A, work,
                                      nbytes, None))
    assert addb(dtype=4) == 2 and addb(dy=None, dsum=None) == 1 and addb(lds=7) == 1
    assert addb(p=-0.5) == 1 and addb(st=None) == 1 and addb(work=None) == 1


def test_refusals_of_the_python_layer(lib):
    from zippel_b200.blocks import rowwise
    x = torch.zeros(2, 8)
    for call in (lambda: rowwise.layer_norm(x), lambda: rowwise.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64)),
                 lambda: rowwise.dropout_add_layer_norm(x, x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        rowwise.layer_norm([1.0, 2.0])
    with pytest.raises(TypeError):
        rowwise.dropout(x, "half", torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        rowwise.ResidualNorm([torch.nn.Linear(8, 8)], 8, p=1.5)
