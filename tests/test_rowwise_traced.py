"""Calls of the operators over rows under torch's tracers, which would keep their result as a constant, and of tensors that
torch wraps without giving them memory: refused."""

from __future__ import annotations

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx


def operators(state):
    from zippel_b200.blocks import rowwise as rw
    return {"layer_norm": lambda v, w: rw.layer_norm(v, w, w), "dropout": lambda v, w: rw.dropout(v, 0.5, state),
            "join": lambda v, w: rw.dropout_add_layer_norm(v, v, w, w, 0.5, state)[0]}


NAMES = sorted(operators(None))


@pytest.fixture(scope="module", params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def device(request):
    if request.param == "cpu":
        from zippel_b200 import build
        build.build_library()
    return request.param


@pytest.mark.parametrize("name", NAMES)
def test_traces_are_refused(device, name):
    """(No device is needed for it, and none spares it.)"""
    state = torch.tensor([1, 2], device=device)
    f = operators(state)[name]
    x, w = torch.randn(4, 8, device=device), torch.ones(8, device=device)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda v: f(v, w) + 2 * v, x, check_trace=False)
    with pytest.raises(RuntimeError, match="trace"):
        make_fx(lambda v: f(v, w) + 2 * v)(x)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_trace_elsewhere_refuses_nothing(name):
    """A trace that is over, and one of another thread."""
    import threading
    f = operators(torch.tensor([1, 2], device="cuda"))[name]
    x, w = torch.randn(4, 8, device="cuda"), torch.ones(8, device="cuda")
    want = f(x, w)
    torch.jit.trace(lambda v: v * 2, x)
    assert torch.equal(f(x, w), want)
    got = []

    def traced(v):
        t = threading.Thread(target=lambda: got.append(f(x, w)))
        t.start()
        t.join()
        return v * 2

    make_fx(traced)(x)
    assert torch.equal(got[0], want)


@pytest.mark.gpu
def test_tensors_without_memory_are_refused():
    """A wrapped weight is not a missing one, nor a wrapped residual or state."""
    from zippel_b200.blocks import rowwise as rw
    x, w = torch.randn(4, 8, device="cuda"), torch.full((8,), 3.0, device="cuda")
    state, wrapped = torch.tensor([1, 2], device="cuda"), torch.func.functionalize
    for call in (lambda: wrapped(lambda v: rw.layer_norm(x, v))(w), lambda: wrapped(lambda v: rw.layer_norm(x, None, v))(w),
                 lambda: wrapped(lambda v: rw.layer_norm(v, w))(x), lambda: wrapped(lambda v: rw.dropout(v, 0.5, state))(x),
                 lambda: wrapped(lambda v: rw.dropout(x, 0.5, v))(state),
                 lambda: wrapped(lambda v: rw.dropout_add_layer_norm(x, v, w, w))(x),
                 lambda: wrapped(lambda v: rw.dropout_add_layer_norm(v, x, w, w)[0])(x),
                 lambda: wrapped(lambda v: rw.dropout_add_layer_norm(x, x, v, w)[0])(w),
                 lambda: wrapped(lambda v: rw.dropout_add_layer_norm(x, x, w, w, 0.5, v)[0])(state)):
        with pytest.raises(RuntimeError, match="no memory of its own"):
            call()
