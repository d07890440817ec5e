"""Which tensors the operators over rows read where they lie and which from a copy: `row_layout` of the extension, on
the CPU.  What is read in place has to be the tensor's own elements, inside its storage."""

from __future__ import annotations

import pytest
import torch

A, B, W = 4, 6, 10


def new(*shape):
    return torch.arange(torch.Size(shape).numel(), dtype=torch.float32).view(*shape)


# name: (tensor, whether it is read from a copy)
LAYOUTS = {
    "dense": (new(A, W), False),
    "dense 3-D": (new(A, B, W), False),
    "one axis": (new(W), False),
    "one number": (new(1)[0], False),
    "rows of a wider array": (new(A, W + 5)[:, 3:3 + W], False),
    "rows of a wider array, 3-D": (new(A, B, W + 5)[..., :W], False),
    "every other row": (new(2 * A, W)[::2], False),
    "one row of a wider array": (new(A, W + 5)[2:3, 1:1 + W], False),
    "axes of one": (new(A, 3, W)[:, 1:2], False),
    "a column": (new(A, W)[:, 3:4], False),
    "some outer rows": (new(A, B, W)[:, 1:4], True),
    "swapped axes": (new(A, B, W).transpose(0, 1), True),
    "transposed": (new(W, A).t(), True),
    "every other element": (new(A, 2 * W)[:, ::2], True),
    "a row repeated": (new(W).expand(A, W), True),
    "a row repeated, as 3-D": (new(W).expand(A, B, W), True),
    "rows repeated inside": (new(A, 1, W).expand(A, B, W), True),
    "rows repeated outside": (new(1, B, W).expand(A, B, W), True),
    "a row repeated once": (new(W).expand(1, W), False),
    "an axis of one, repeated rows": (new(A, 1, 1, W).expand(A, 1, B, W), True),
    "a number repeated": (new(1, 1).expand(A, W), True),
    "a number repeated, one column": (new(1, 1).expand(A, 1), True),
    "a number repeated, one column, 3-D": (new(A, 1, 1).expand(A, B, 1), True),
    "rows that overlap": (new(64).as_strided((A, W), (3, 1)), True),
    "rows that overlap, outside": (new(64).as_strided((2, 3, W), (W, W, 1)), True),
    "rows that overlap, inside": (new(64).as_strided((2, 3, W), (30, 5, 1)), True),
    "no rows": (new(A, W)[:0, :3], None),
    "no columns": (new(A, W)[:, :0], None),
}


@pytest.fixture(scope="module")
def row_layout():
    from zippel_b200 import build
    build.build_library()
    from zippel_b200 import _rowwise
    return _rowwise.row_layout


def check(row_layout, x, copied):
    rows, width, ld, took_copy = row_layout(x)
    assert width == (x.shape[-1] if x.dim() else 1) and rows == (x.numel() // width if width else 0)
    assert ld >= width
    if x.numel() == 0:
        return
    assert copied is None or took_copy == copied
    if not took_copy:                          # (as_strided refuses what lies outside the storage)
        read = x.as_strided((rows, width), (ld, 1), x.storage_offset())
        assert torch.equal(read, x.reshape(rows, width))


@pytest.mark.parametrize("name", LAYOUTS)
def test_rows_that_are_read_in_place_are_the_tensors_own(row_layout, name):
    check(row_layout, *LAYOUTS[name])


@pytest.mark.parametrize("sum_over", [0, 1, (0, 1), (0, 1, 2)])
@pytest.mark.parametrize("shape", [(A, B, W), (A, B, 1), (1, B, W), (A, 1, W)])
def test_gradients_of_sums(row_layout, shape, sum_over):
    """What autograd hands over for the sum of a result: expanded tensors."""
    seen = []

    class Result(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            seen.append(g)
            return g

    y = Result.apply(new(*shape).requires_grad_())
    (y.sum(sum_over) ** 2).sum().backward()
    check(row_layout, seen[0], None)


def test_random_strides(row_layout):
    """Views of every kind of stride, zeroes among them, over one storage."""
    g = torch.Generator().manual_seed(0)
    pick = lambda *of: of[int(torch.randint(len(of), (), generator=g))]             # noqa: E731
    base = new(4096)
    for _ in range(3000):
        dims = pick(1, 2, 3, 4)
        shape = [pick(1, 2, 3, 5) for _ in range(dims)]
        dense, strides = 1, []
        for n in reversed(shape):              # the dense stride, none, or another
            strides.insert(0, pick(dense, dense, dense, 0, 1, 2, dense + 3))
            dense = max(strides[0], 1) * n if pick(0, 0, 1) == 0 else dense * n
        if 7 + sum((n - 1) * s for n, s in zip(shape, strides)) >= base.numel():
            continue
        check(row_layout, base.as_strided(shape, strides, 7), None)


def lazy_tensors():
    z = torch.complex(new(A, W), -new(A, W)).conj()
    return {"negated": torch._neg_view(new(A, W)), "negated, one axis": torch._neg_view(new(W)),
            "a column of imaginary parts": z[:, :1].imag, "an imaginary part": z[:1, :1].imag,
            "imaginary parts": z.imag, "negated rows of a wider array": torch._neg_view(new(A, W + 5)[:, :W]),
            "zeroes that are not stored": torch._efficientzerotensor((A, W))}


@pytest.mark.parametrize("name", lazy_tensors())
def test_values_that_are_not_in_memory_come_from_a_copy(row_layout, name):
    """Lazy negations and zeroes without storage: what lies at the tensor's address is not its values."""
    x = lazy_tensors()[name]
    rows, width, ld, copied = row_layout(x)
    assert copied and (rows, width) == (x.numel() // x.shape[-1], x.shape[-1]) and ld >= width
